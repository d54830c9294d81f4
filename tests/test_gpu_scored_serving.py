"""Serving with attention over the paged cache and scored answers (GPU).

The engine, colocated and disaggregated, with the model's layers attending through
iekv_attend: greedy output must be that of the torch path, whatever the cache type, the
window and the prefixes its requests share. Every generated token's score must be that of
the logits it was drawn from.

The scores' tolerance: logits of the toy model lie within 32, so a difference from the
largest, its exponential and the logarithm of the sum are each off by at most a few steps of
a number below 64 (2^-18), the sum of 256 terms by 256 2^-24 relative to itself.
"""
from __future__ import annotations

import pytest
import torch

from conftest import golden

pytestmark = pytest.mark.gpu

G = golden("disaggregation")
TYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn]


def model(device, cache_dtype=torch.float32, **options):
    from iekv.engine.toy_model import ModelConfig, ToyTransformer

    return ToyTransformer(ModelConfig(**G["model"]), seed=G["model_seed"], device=device,
                          cache_dtype=cache_dtype, **options)


def engine_config(**over):
    from iekv.engine.engine import EngineConfig

    return EngineConfig(**{**G["engine"], **over})


def decided(device, prompts, n, **options):
    """Greedy tokens of the torch path, up to the first that rounding could decide: the
    model's logits, of size one, are off by some 1e-5 in 32 bits, and its two best ones have
    come within 1e-5 of each other."""
    from iekv.engine.engine import Engine

    toy, rows, outs = model(device, **options), [], []
    whole = toy.last_token_logits

    def recorded(hidden, query_lens):
        rows.append(whole(hidden, query_lens).cpu())
        return rows[-1]

    toy.last_token_logits = recorded
    for prompt in prompts:
        rows.clear()
        tokens = Engine(toy, engine_config()).generate([prompt], max_new_tokens=n,
                                                       temperature=0.0)[0]
        best = torch.cat(rows)[-n:].topk(2, 1).values
        close = (best[:, 0] - best[:, 1] < 1e-4).tolist()
        outs.append(tokens[:close.index(True) if True in close else n])
    return outs


@pytest.mark.parametrize("cache_dtype", TYPES, ids=str)
@pytest.mark.parametrize("window, sinks", [(None, 0), (9, 2)])
def test_the_model_decodes_identically_through_paged_attention(gpu, cache_dtype, window, sinks):
    from iekv.engine.engine import Engine
    from iekv.serve.disaggregated import DisaggregatedEngine

    options = dict(cache_dtype=cache_dtype, window=window, sinks=sinks)
    # torch scatters no 8-bit rows: there the slot kernels do on either side.
    only = [True] if cache_dtype == torch.float8_e4m3fn else [False, True]
    want = decided(gpu, G["prompts"], 8, hip_kv=only[0], **options)
    assert sum(map(len, want)) > 4 * len(want)
    for hip_kv in only:
        hip = model(gpu, hip_kv=hip_kv, hip_attention=True, **options)
        for engine in (Engine(hip, engine_config()),
                       DisaggregatedEngine(hip, engine_config(), mode="direct")):
            got = engine.generate(G["prompts"], max_new_tokens=8, temperature=0.0)
            assert [g[:len(w)] for g, w in zip(got, want)] == want


def test_a_window_changes_what_is_decoded_and_sinks_do_too(gpu):
    from iekv.engine.engine import Engine

    outs = []
    for window, sinks in ((None, 0), (3, 0), (3, 2)):
        hip = model(gpu, hip_attention=True, window=window, sinks=sinks)
        layers = Engine(hip, engine_config())
        outs.append(layers.generate(G["prompts"], max_new_tokens=12, temperature=0.0))
    assert outs[0] != outs[1] and outs[1] != outs[2]


def test_requests_behind_one_prefix_attend_it_once(gpu, monkeypatch):
    """Requests that share the first blocks of one that came before them: the plans of the
    decode steps say so, and the output is that of the torch path."""
    from iekv.engine import attention
    from iekv.engine.engine import Engine

    bs = G["engine"]["block_size"]
    prefix = [(7 * i + 3) % G["model"]["vocab_size"] for i in range(4 * bs)]
    prompts = [prefix + [11 + i, 5 + 2 * i] for i in range(5)]
    config = engine_config(num_blocks=256)
    want = Engine(model(gpu), config).generate(prompts, max_new_tokens=6, temperature=0.0)
    seen = []
    common = attention.common_blocks

    def spy(tables, contexts, block_size):
        seen.append(common(tables, contexts, block_size))
        return seen[-1]

    monkeypatch.setattr(attention, "common_blocks", spy)
    engine = Engine(model(gpu, hip_kv=True, hip_attention=True), config)
    seqs = [engine.submit(prompts[0], max_new_tokens=6, temperature=0.0)]
    engine.step()                       # its blocks are there to be shared
    seqs += [engine.submit(p, max_new_tokens=6, temperature=0.0) for p in prompts[1:]]
    engine.run()
    assert [s.token_ids[s.num_prompt:] for s in seqs] == want
    assert max(seen) >= 4


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_scores_are_those_of_the_logits(gpu, temperature):
    from iekv.engine.engine import Engine

    class Recording(type(model(gpu))):
        rows = []

        def last_token_logits(self, hidden, query_lens):
            logits = super().last_token_logits(hidden, query_lens)
            self.rows.append(logits.double().cpu())
            return logits

    from iekv.engine.toy_model import ModelConfig

    hip = Recording(ModelConfig(**G["model"]), seed=G["model_seed"], device=gpu, hip_kv=True,
                    hip_attention=True)
    Recording.rows = []
    engine, done = Engine(hip, engine_config(logprobs=3)), []
    for prompt in G["prompts"]:                # one after the other: rows in their order
        engine.submit(prompt, max_new_tokens=5, temperature=temperature)
        done += engine.run()
    assert len(done) == len(G["prompts"])
    scored = [s for seq in done for s in seq.scores]
    generated = [t for seq in done for t in seq.token_ids[seq.num_prompt:]]
    assert [s.token_id for s in scored] == generated
    tol = 8 * 2.0 ** -18 + 256 * 2.0 ** -24
    assert all(len(seq.scores) == seq.num_generated for seq in done)
    # A chunk of a prompt leaves a row without a token.
    rows = iter(torch.cat(Recording.rows))
    for score in scored:
        for row in rows:
            assert row.abs().max() < 32
            lp = torch.log_softmax(row, 0)
            entropy = -(lp.exp() * lp).sum()
            if abs(lp[score.token_id] - score.logprob) <= tol and \
                    abs(entropy - score.entropy) <= 16 * tol:
                break
        else:
            pytest.fail(f"no row scores token {score.token_id} with {score.logprob}")
        order = torch.sort(row.float(), descending=True, stable=True).indices[:3].tolist()
        assert [t for t, _ in score.top] == order
        assert all(abs(lp[t] - v) <= tol for t, v in score.top)


def test_scores_move_with_a_handoff(gpu):
    from iekv.engine.engine import Engine
    from iekv.serve.disaggregated import DisaggregatedEngine

    prompt = G["prompts"][0]
    colocated = Engine(model(gpu, hip_attention=True), engine_config(logprobs=2))
    alone = colocated.submit(prompt, max_new_tokens=6, temperature=0.0)
    colocated.run()
    split = DisaggregatedEngine(model(gpu, hip_attention=True), engine_config(logprobs=2),
                                mode="direct")
    transfer = split.prefill.prefill(prompt, 0.0)
    assert len(transfer.scores) == 1
    seq = split.decode.admit(transfer, 6, 0.0)
    split.decode.engine.run()
    assert seq.token_ids == alone.token_ids
    assert [s.token_id for s in seq.scores] == seq.token_ids[seq.num_prompt:]
    assert len(seq.scores) == len(alone.scores)
    for a, b in zip(seq.scores, alone.scores):
        assert abs(a.logprob - b.logprob) < 1e-4 and [t for t, _ in a.top] == [t for t, _ in b.top]
