"""Scores of generated tokens over the wire (GPU)."""
from __future__ import annotations

import pytest

from test_gpu_scored_serving import G, engine_config, model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", ["pack", "direct"])
def test_scores_over_the_wire_are_those_of_one_engine(gpu, mode):
    from iekv.engine.engine import Engine
    from iekv.serve.disaggregated import DisaggregatedEngine
    from iekv.serve.wire import from_wire, to_wire

    m = model(gpu, hip_attention=True)
    split = DisaggregatedEngine(m, engine_config(logprobs=2), mode=mode)
    for prompt in G["prompts"][:3]:
        colocated = Engine(m, engine_config(logprobs=2))
        alone = colocated.submit(prompt, max_new_tokens=6, temperature=0.0)
        colocated.run()
        header, payload = to_wire(split.prefill.prefill(prompt))
        seq = split.decode.admit(from_wire(header, payload.clone()), 6, 0.0)
        split.decode.engine.run()
        generated = seq.token_ids[seq.num_prompt:]
        assert seq.token_ids == alone.token_ids
        assert [s.token_id for s in seq.scores] == generated and len(generated) == 6
        for a, b in zip(seq.scores, alone.scores):
            assert abs(a.logprob - b.logprob) < 1e-4 and abs(a.entropy - b.entropy) < 1e-3
            assert [t for t, _ in a.top] == [t for t, _ in b.top]
