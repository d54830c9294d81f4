"""Scores of generated tokens on their way through handoffs (CPU; the scoring itself is in
test_gpu_scored_serving.py)."""
from __future__ import annotations

import math

import pytest

from test_engine import engine
from test_wire import make_transfer, packed_from_oracle


def score(token, logprob=-0.5):
    from iekv.engine.engine import TokenScore

    return TokenScore(token, logprob, 1.25, [(token, logprob), (7, -2.0)])


def test_scores_go_over_the_wire():
    from iekv.serve.wire import decode_header, from_wire, to_wire

    packed, _ = packed_from_oracle()
    transfer = make_transfer(packed)
    plain, payload = to_wire(transfer)
    assert "scores" not in decode_header(plain)          # as it was where nothing is scored
    assert from_wire(plain, payload.clone()).scores == []
    transfer.scores = [score(130), None, score(9, -math.inf), score(3, math.nan)]
    header, payload = to_wire(transfer)
    assert b"NaN" not in header and b"Infinity" not in header     # JSON has no such numbers
    back = from_wire(header, payload.clone()).scores
    assert back[:3] == transfer.scores[:3]
    assert back[3].token_id == 3 and math.isnan(back[3].logprob) and \
        math.isnan(back[3].top[0][1]) and back[3].top[1] == (7, -2.0)


def workers():
    """Prefill and decode engines over the reference's copier, whose decode engine scores as
    if a GPU did."""
    from iekv.engine.toy_model import ModelConfig, ToyTransformer
    from iekv.engine.engine import EngineConfig
    from iekv.serve.disaggregated import DisaggregatedEngine
    from test_engine import SMALL, oracle_factory

    model = ToyTransformer(ModelConfig(**SMALL), seed=0, device="cpu")
    both = DisaggregatedEngine(model, EngineConfig(block_size=8, num_blocks=64),
                               copier_factory=oracle_factory)
    return both, both.prefill, both.decode


def scoring(engine, monkeypatch):
    monkeypatch.setattr(engine.config, "logprobs", 2)
    monkeypatch.setattr(engine, "_score", lambda logits, tokens: [score(t) for t in tokens])


@pytest.mark.parametrize("new_tokens", [1, 5])
def test_scores_keep_their_tokens_when_the_first_was_not_scored(monkeypatch, new_tokens):
    """The prefill worker was not asked to score (or its scores were lost on the way): entry i
    is still that of generated token i."""
    both, prefill, decode = workers()
    transfer = prefill.prefill([3, 1, 4, 1, 5, 9, 2, 6], 0.0)
    assert transfer.scores == []
    scoring(decode.engine, monkeypatch)
    seq = decode.admit(transfer, new_tokens, 0.0)
    both.decode_until_done()
    generated = seq.token_ids[seq.num_prompt:]
    assert len(generated) == new_tokens == len(seq.scores)
    assert seq.scores[0] is None
    assert [s.token_id for s in seq.scores[1:]] == generated[1:]


def test_an_engine_that_is_asked_late_scores_the_tokens_it_is_asked_for(monkeypatch):
    eng = engine()
    seq = eng.submit([1, 2, 3], max_new_tokens=5, temperature=0.0)
    eng.step()
    eng.step()
    scoring(eng, monkeypatch)
    eng.run()
    generated = seq.token_ids[seq.num_prompt:]
    assert seq.scores[:2] == [None, None]
    assert [s.token_id for s in seq.scores[2:]] == generated[2:]


def test_scores_of_a_prefill_stay_where_decode_does_not_score(monkeypatch):
    both, prefill, decode = workers()
    transfer = prefill.prefill([3, 1, 4, 1, 5], 0.0)
    transfer.scores = [score(transfer.token_ids[-1])]
    seq = decode.admit(transfer, 3, 0.0)
    both.decode_until_done()
    assert [s.token_id for s in seq.scores] == [seq.token_ids[seq.num_prompt]]


@pytest.mark.parametrize("logprobs, said", [
    (65, "at most 64"), (-1, "logprobs -1"), (33, "vocabulary of 32"), (3, "on cpu")])
def test_engines_refuse_what_no_step_could_be_scored_with(logprobs, said):
    """Before anything is scheduled: a step that raises has computed and committed nothing."""
    from iekv.engine.engine import Engine, EngineConfig
    from iekv.engine.toy_model import ModelConfig, ToyTransformer
    from test_engine import SMALL

    model = ToyTransformer(ModelConfig(**dict(SMALL, vocab_size=32)), seed=0, device="cpu")
    with pytest.raises(ValueError, match=said):
        Engine(model, EngineConfig(block_size=8, num_blocks=16, logprobs=logprobs))


def test_scores_are_of_the_logits_that_forward_returned(monkeypatch):
    """An engine whose forward changes the logits, and a model that has no logits but
    those forward takes from it."""
    import numpy as np

    from iekv.engine.engine import Engine

    seen = []

    class Barring(Engine):
        def forward(self, batch):
            layout, logits = super().forward(batch)
            logits = logits.copy()
            logits[:, ::2] = -np.inf
            return layout, logits

    eng = engine()
    eng.__class__ = Barring
    monkeypatch.delattr(type(eng.model), "last_token_logits")
    monkeypatch.setattr(type(eng.model), "logits_for_last_token_of_each",
                        lambda self, hidden, lens: np.tile(
                            np.arange(64, dtype=np.float32), (len(lens), 1)))
    monkeypatch.setattr(eng.config, "logprobs", 2)
    monkeypatch.setattr(eng, "_score", lambda logits, tokens: seen.append(logits) or
                        [score(t) for t in tokens])
    seq = eng.submit([1, 2, 3], max_new_tokens=3, temperature=0.0)
    eng.run()
    assert seq.token_ids[3:] == [63, 63, 63] and len(seq.scores) == 3
    assert all(np.isneginf(x[:, ::2]).all() and (x[:, 1] == 1).all() for x in seen)
