"""Decoders whose vocabulary or hidden width is below the tensor-core tile's 16 columns, so that some
of a step's projections take the tiled or GEMV kernels beside others on the tensor cores."""
import numpy as np
import pytest

from basalt_b200 import ModelSpec, left_pad, synthetic_prompts
from parity import compare_logits
from test_gpu_decoder import make_pair

pytestmark = pytest.mark.gpu


def check(runtime, path, spec, rows, prompt, steps):
    engine, oracle = make_pair(runtime, spec, path, seed=rows, stddev=0.1)
    contexts = left_pad(synthetic_prompts(rows, rows, prompt, spec.vocabulary), spec.window, spec.vocabulary)
    tokens, logits = engine.generateWithLogits(contexts, steps)
    for r in range(0, rows, max(1, rows // 24)):
        compare_logits(logits[r], oracle.forced_scores(contexts[r], tokens[r]), where=f"row {r}")
    engine.close()


@pytest.mark.parametrize("vocabulary,dim,heads,hidden", [(5, 256, 2, 64), (15, 96, 3, 256), (97, 256, 4, 8),
                                                         (9, 512, 4, 8), (16, 256, 4, 16)])
@pytest.mark.parametrize("rows", [9, 16])
@pytest.mark.parametrize("kw", [{}, {"weight_dtype": "bf16"}, {"attention_window": 40}])
def test_split_projections_feed_ones_without_operand_planes(runtime, tmp_path, vocabulary, dim, heads, hidden,
                                                            rows, kw):
    check(runtime, tmp_path / "w.bin", ModelSpec("padded_decoder", vocabulary, 40, dim, 2, heads, hidden,
                                                 **kw), rows, 6, 8)


@pytest.mark.parametrize("vocabulary,dim,heads,hidden", [(5, 128, 2, 64), (15, 96, 3, 48), (5, 64, 1, 24),
                                                         (97, 64, 2, 8), (9, 256, 4, 8)])
@pytest.mark.parametrize("rows", [18, 33, 200])
def test_rows_in_lanes_keep_their_own_normalised_inputs(runtime, tmp_path, vocabulary, dim, heads, hidden,
                                                        rows):
    check(runtime, tmp_path / "w.bin", ModelSpec("padded_decoder", vocabulary, 40, dim, 2, heads, hidden),
          rows, 6, 8)
