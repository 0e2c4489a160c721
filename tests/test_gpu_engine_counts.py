"""What an engine counts of the attention that it runs through the serving operators."""
import pytest

from basalt_b200 import ModelSpec, TextEngine, left_pad, synthetic_prompts, write_synthetic_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("storage,value_bytes", [("u4", 0.625), ("bf16", 2), ("f32", 4)])
@pytest.mark.parametrize("context,prompt,kernels", [(700, 600, 2), (40, 20, 1)])
def test_launches_and_bytes_of_a_step(runtime, tmp_path, storage, value_bytes, context, prompt, kernels):
    """600 keys of two heads are split over CTAs and joined by a second kernel, 25 are not."""
    V, L, H, D, steps = 30, 2, 2, 64, 5
    spec = ModelSpec("padded_decoder", V, context, D, L, H, 64, kv_dtype=storage, attention_window=context)
    write_synthetic_weights(spec, tmp_path / "w.bin", seed=1)
    engine = TextEngine.of(runtime, spec, V, context)
    engine.load(tmp_path / "w.bin")
    contexts = left_pad(synthetic_prompts(1, 1, prompt, V), context, V)
    engine.generateBatch(contexts, steps)
    engine.profile()
    engine.profile_reset()
    engine.generateBatch(contexts, 1)
    before = {k: dict(v) for k, v in engine.profile_read().items()}
    engine.profile_reset()
    engine.generateBatch(contexts, steps)
    after = engine.profile_read()
    engine.profile(False)
    engine.close()
    decode = steps - 1
    assert after["attn_decode"]["launches"] == decode * L * kernels
    # a step stores one token's keys and values in every layer, from float32
    stored = after["misc"]["bytes"] - before["misc"]["bytes"]
    assert stored == decode * L * 2 * D * (4 + value_bytes)
