"""Serving from microscaled caches (GPU): the toy model's rows are quantised as they are written
and attended over, colocated and after a handoff, from the offload tier and over the wire."""
from __future__ import annotations

import pytest
import torch

from quantized_reference import FORMATS, decode, encode
from test_gpu_scored_serving import G, decided, engine_config, model

pytestmark = pytest.mark.gpu


def agree(got, want):
    assert [g[:len(w)] for g, w in zip(got, want)] == want


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("window, sinks", [(None, 0), (9, 2)])
def test_the_model_decodes_alike_on_every_path(gpu, format, window, sinks):
    """Contexts that are read back and attended in torch, attention over the records, and a
    handoff of the records between the two workers: the same tokens."""
    from iekv.engine.engine import Engine
    from iekv.serve.disaggregated import DisaggregatedEngine

    options = dict(cache_format=format, window=window, sinks=sinks)
    want = decided(gpu, G["prompts"], 8, hip_kv=True, **options)
    assert sum(map(len, want)) > 4 * len(want)
    for m in (model(gpu, hip_attention=True, **options),
              model(gpu, hip_kv=True, hip_attention=True, **options),
              model(gpu, hip_kv=True, **options)):
        for engine in (Engine(m, engine_config()), DisaggregatedEngine(m, engine_config()),
                       DisaggregatedEngine(m, engine_config(), mode="direct"),
                       DisaggregatedEngine(m, engine_config(), mode="queue")):
            agree(engine.generate(G["prompts"], max_new_tokens=8, temperature=0.0), want)


@pytest.mark.parametrize("format", FORMATS)
def test_the_caches_hold_what_the_formats_make_of_the_rows(gpu, format):
    """Of the first layer, whose rows no attention comes before."""
    from iekv.engine.engine import Engine

    prompt = G["prompts"][0]
    plain = Engine(model(gpu), engine_config())
    scaled = Engine(model(gpu, hip_attention=True, cache_format=format), engine_config())
    tables = []
    for engine in (plain, scaled):
        seq = engine.submit(prompt, max_new_tokens=4, temperature=0.0)
        engine.step()
        tables.append(list(seq.block_table))
    assert tables[0] == tables[1]
    bs = plain.config.block_size
    rows = [tables[0][j // bs] * bs + j % bs for j in range(len(prompt))]
    for a, b in ((plain.k_caches, scaled.k_caches), (plain.v_caches, scaled.v_caches)):
        want = decode(encode(a[0][rows], format), format)
        assert torch.equal(decode(b[0][rows], format), want)


@pytest.mark.parametrize("over", [dict(offload_blocks=64, num_blocks=24),
                                  dict(preemption="swap", num_blocks=24)], ids=["tier", "swap"])
def test_records_come_back_from_host_memory(gpu, over):
    from iekv.engine.engine import Engine

    m = model(gpu, hip_kv=True, hip_attention=True, cache_format="mxint8")
    want = Engine(m, engine_config()).generate(G["prompts"], max_new_tokens=8, temperature=0.0)
    engine = Engine(m, engine_config(**over))
    for _ in range(2):                       # the second time behind resident or offloaded blocks
        got = engine.generate(G["prompts"], max_new_tokens=8, temperature=0.0)
        close = sum(g != w for g, w in zip(got, want))
        assert close <= 1                    # a token that rounding could decide


def test_records_travel_over_the_wire(gpu):
    from iekv.serve.disaggregated import DecodeWorker, PrefillWorker
    from iekv.serve.wire import from_wire, to_wire

    m = model(gpu, hip_attention=True, cache_format="mxfp8")
    prefill, decode_side = PrefillWorker(m, engine_config()), DecodeWorker(m, engine_config())
    prompt = G["prompts"][1]
    transfer = prefill.prefill(prompt, 0.0)
    header, payload = to_wire(transfer)
    back = from_wire(header, payload.cpu())
    seq = decode_side.admit(back, max_new_tokens=6, temperature=0.0)
    n, bs = len(prompt), prefill.engine.config.block_size
    sent = payload.cpu()
    for index, block in enumerate(seq.block_table[:n // bs]):
        for a, cache in enumerate(decode_side.engine.k_caches + decode_side.engine.v_caches):
            assert torch.equal(cache[block * bs:(block + 1) * bs].cpu().view(-1), sent[index, a])
    decode_side.engine.run()
    want = decided(gpu, [prompt], 6, hip_kv=True, cache_format="mxfp8")
    agree([seq.token_ids[seq.num_prompt:]], want)


def test_models_without_the_slot_kernels_are_refused(gpu):
    with pytest.raises(ValueError, match="hip_kv or hip_attention"):
        model(gpu, cache_format="mxfp8")
    with pytest.raises(ValueError, match="no format"):
        model(gpu, hip_kv=True, cache_format="fp8")


def pools_of(format, other, dim=32):
    """Two registered pools of the same bytes in records of `format` and of `other` (None: bytes)."""
    from iekv.engine.copier import HipSlotCopier
    from iekv.engine.quantized import allocate_quantized_pool

    made = []
    for f in (format, other):
        k, v = allocate_quantized_pool(6, 4, 2, 2, dim, format="mxfp8")
        made.append(HipSlotCopier(k, v, 4, format=f))
    return made


@pytest.mark.parametrize("format, other", [("mxfp8", "mxint8"), ("mxint8", "mxfp8"),
                                           ("mxfp8", None), (None, "mxint8")])
def test_blocks_do_not_go_where_another_format_is(gpu, format, other):
    """The records of both are of one size: nothing but the format tells them apart."""
    from iekv.engine.quantized import QuantizedPool
    from iekv.engine.queue import HandoffQueue

    source, destination = pools_of(format, other)
    for t in source.k_caches + source.v_caches:
        t.fill_(7)
    refused = pytest.raises(ValueError, match="records")
    with refused:
        destination.copy_blocks(source, [0, 1], [2, 3])
    with refused:
        destination.copy_requests(source, [([0, 1], [2, 3])])
    with pytest.raises(ValueError, match="what they hold"):
        HandoffQueue(source.pool, destination.pool)
    for location in ("device", "host"):
        packed = source.read_blocks([0, 1, 4], location=location)
        for payloads in (packed, [packed[2], packed[0]], packed[::2]):
            with refused:
                destination.write_blocks([1, 2, 3][:len(payloads)], payloads)
        with refused:
            destination.read_blocks([1, 2, 3], into=source.empty_payloads(3))
    torch.cuda.synchronize()
    assert not any(t.any() for t in destination.k_caches + destination.v_caches)
    for f, copier in ((format, source), (other, destination)):
        if f is not None:
            pool = QuantizedPool(copier.k_caches, copier.v_caches, 4, f)
            assert pool.same_shape(copier.pool) and copier.pool.same_shape(pool)
    # Of one format, as ever.
    destination.format = format
    destination.copy_blocks(source, [0], [2])
    destination.write_blocks([3], source.read_blocks([1]))
    torch.cuda.synchronize()
    for t in destination.k_caches + destination.v_caches:
        assert t.view(6, -1)[2:4].eq(7).all() and not t.view(6, -1)[[0, 1, 4, 5]].any()


def test_a_copiers_format_is_one_that_its_caches_can_hold(gpu):
    source, _ = pools_of("mxfp8", None)
    with pytest.raises(ValueError, match="no format"):
        source.format = "mxfp6"
    with pytest.raises(ValueError, match="none of mxfp4"):       # that would be heads of 144
        pools_of("mxfp8", None, dim=72)[0].format = "mxfp4"
    assert source.format == "mxfp8"


@pytest.mark.parametrize("mode", ["pack", "direct", "queue"])
def test_a_worker_refuses_transfers_of_another_format(gpu, mode):
    from iekv.serve.disaggregated import DecodeWorker, PrefillWorker
    from iekv.serve.wire import from_wire, to_wire

    prefill = PrefillWorker(model(gpu, hip_attention=True, cache_format="mxfp8"), engine_config(),
                            mode=mode)
    worker = DecodeWorker(model(gpu, hip_attention=True, cache_format="mxint8"), engine_config())
    worker.use_queue = mode == "queue"
    free = worker.engine.blocks.num_free
    transfer = prefill.prefill(G["prompts"][1], 0.0)
    with pytest.raises(ValueError, match="transfer of mxfp8, .* hold mxint8"):
        worker.admit(transfer, max_new_tokens=4)
    with pytest.raises(ValueError, match="transfer of mxfp8, .* hold mxint8"):
        worker.admit(from_wire(*to_wire(transfer)), max_new_tokens=4)
    assert worker.engine.blocks.num_free == free and not worker.engine.scheduler.waiting


def watched_copier():
    """A copier that compares what it moves to and from host memory with the pool's bytes."""
    from iekv.engine.copier import HipSlotCopier

    class Watched(HipSlotCopier):
        out = back = 0

        def same(self, block_ids, images):
            torch.cuda.synchronize()
            for block, image in zip(block_ids, images, strict=True):
                rows = slice(block * self.block_size, (block + 1) * self.block_size)
                for a, cache in enumerate((*self.k_caches, *self.v_caches)):
                    assert torch.equal(cache[rows].cpu().view(-1), image[a])

        def read_blocks(self, block_ids, **kw):
            packed = super().read_blocks(block_ids, **kw)
            assert packed.on_host and packed.format == self.format is not None
            self.same(block_ids, packed.host_data())
            self.out += len(packed)
            return packed

        def _offload_each(self, block_ids, payloads):
            super()._offload_each(block_ids, payloads)
            self.same(block_ids, [p.packed.host_data()[p.index] for p in payloads])
            self.out += len(payloads)

        def write_blocks(self, block_ids, payloads, **kw):
            images = [p.packed.host_data()[p.index].clone() for p in payloads]
            super().write_blocks(block_ids, payloads, **kw)
            self.same(block_ids, images)
            self.back += len(images)

    return lambda k, v, block_size, role: Watched(k, v, block_size, payload_location="host",
                                                  defer_reads=role == "offload")


# Pools that hold two of four prompts: the second time behind offloaded blocks, and requests that
# grow past the pool while they decode.
PRESSED = {"tier": (dict(offload_blocks=64, num_blocks=8), 48, 8),
           "swap": (dict(block_size=8, num_blocks=8, preemption="swap"), 12, 10)}


@pytest.mark.parametrize("where", list(PRESSED))
@pytest.mark.parametrize("format", FORMATS)
def test_records_go_to_host_memory_and_come_back(gpu, format, where):
    from iekv.engine.engine import Engine

    over, length, n = PRESSED[where]
    prompts = [p[:length] for p in G["prompts"]]
    want = decided(gpu, prompts, n, hip_kv=True, cache_format=format)
    assert sum(map(len, want)) > 4 * len(want)
    m = model(gpu, hip_kv=True, hip_attention=True, cache_format=format)
    engine = Engine(m, engine_config(**over), copier_factory=watched_copier())
    for _ in range(2):
        agree(engine.generate(prompts, max_new_tokens=n, temperature=0.0), want)
    if where == "tier":
        assert engine.blocks.tier.stats.restored == engine.copier.back > 0
        assert engine.copier.out >= engine.copier.back
    else:
        stats = engine.scheduler.stats
        assert stats.swapped_in == stats.swapped_out > 0
        assert engine.swapper.out == engine.swapper.back > 0
