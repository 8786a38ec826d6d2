"""Steps of the engine that bring a portion and single tokens at once, over a cache of 8 bits, against the decoder from its formulas in 64 bits."""

from __future__ import annotations

import pytest
import torch

import tiny_configs
from liteinfer_b200.engine.loading import build_runner
from liteinfer_b200.engine.runner import StepEntry
from test_int8_engine_gpu import PlainInt8Llama, _off

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("name", ["tiny_d", "tiny_e"])
def test_portions_beside_single_tokens(model_dirs, name, weights, graphs):
    """Two requests decode while a third's prompt comes in portions, in graphs of padded shapes and kernel by kernel (the bounds are those of
    the engine's other steps in 32 bits: 0.5 % with the cache alone in 8 bits, 8 % with the products' roundings)."""
    bound = 8e-2 if weights else 5e-3
    config, _, page = tiny_configs.ALL[name]
    runner = build_runner(model_dirs[name], torch.float32, "cuda:0", page, 120, 4, int8_weights=weights, int8_cache=True)
    if graphs:
        runner.enable_decode_graphs(4, 512)
    vocab = config["vocab_size"]
    prompts = [tiny_configs.prompt(vocab, n, i) for i, n in enumerate((61, 16, 150))]
    forced = [tiny_configs.prompt(vocab, 12, 10 + i) for i in range(3)]
    plain = [PlainInt8Llama(model_dirs[name], page, weights, True) for _ in range(3)]
    got = runner.step([StepEntry("a", prompts[0], (60,)), StepEntry("b", prompts[1], (15,))])
    for row, p, prompt in zip(got, plain, prompts):
        assert _off(row, p.step(prompt)[-1]) <= bound
    cuts, at = [40, 1, 70, 2, 37], 0
    for t, cut in enumerate(cuts):
        portion = prompts[2][at:at + cut]
        at += cut
        got = runner.step([StepEntry("a", [forced[0][t]], (0,)), StepEntry("c", portion, tuple(range(cut))), StepEntry("b", [forced[1][t]], (0,))])
        assert _off(got[0], plain[0].step([forced[0][t]])[0]) <= bound
        assert _off(got[1:1 + cut], plain[2].step(portion)) <= bound
        assert _off(got[1 + cut], plain[1].step([forced[1][t]])[0]) <= bound
    assert at == 150
    assert (runner.graph_replays > 0) == graphs
    runner.check_kernels()
