"""What caches hold travels with their blocks (CPU): payloads, the wire's header and the decode
worker's admission carry the format of microscaled records, of which two may have the same size."""
from __future__ import annotations

import json

import pytest
import torch

from helpers import oracle_factory
from test_disaggregation import engine_config, model
from test_wire import make_transfer


def packed_of(format, record=36, blocks=3, layers=2, bs=4, heads=2):
    from iekv.engine.copier import PackedBlocks

    data = torch.arange(blocks * 2 * layers * bs * heads * record, dtype=torch.int64) % 251
    return PackedBlocks(data.to(torch.uint8).view(blocks, 2 * layers, -1), layers,
                        (bs, heads, record), torch.uint8, format)


@pytest.mark.parametrize("format", ["mxfp8", "mxint8", "mxfp4", None])
def test_the_format_is_in_the_header(format):
    from iekv.serve.wire import decode_header, from_wire, to_wire

    packed = packed_of(format)
    assert packed[1:].format == packed[0].packed.format == format
    header, payload = to_wire(make_transfer(packed))
    meta = decode_header(header)
    assert meta.get("cache_format") == format
    assert ("cache_format" in meta) == (format is not None)     # values: as it was
    back = from_wire(header, payload.clone()).block_payloads
    assert back.format == format and torch.equal(back.data, packed.data)
    transfer = make_transfer(packed)
    transfer.block_payloads = [packed[2], packed[0]]
    assert from_wire(*to_wire(transfer)).block_payloads.format == format


@pytest.mark.parametrize("said", ["mxfp6", 5, ["mxfp8"], False])
def test_formats_that_are_not_known_are_refused(said):
    from iekv.serve.wire import _PREFIX, decode_header, encode_header

    header = encode_header(make_transfer(packed_of("mxfp8")), packed_of("mxfp8"))
    magic, version, _ = _PREFIX.unpack_from(header)
    meta = json.loads(header[_PREFIX.size:])
    meta["cache_format"] = said
    body = json.dumps(meta).encode()
    with pytest.raises(ValueError, match="unknown cache format"):
        decode_header(_PREFIX.pack(magic, version, len(body)) + body)


@pytest.mark.parametrize("a, b", [("mxfp8", "mxint8"), ("mxfp8", None), (None, "mxint8")])
def test_payloads_of_two_formats_are_not_put_together(a, b):
    from iekv.engine.copier import stack_payloads

    with pytest.raises(ValueError, match=a or b):
        stack_payloads([packed_of(a)[0], packed_of(b)[0]])
    assert stack_payloads([packed_of(a)[0], packed_of(a)[2]]).format == a


def tagged(format):
    """Copiers that know what they move, as HipSlotCopier does."""
    def factory(k_caches, v_caches, block_size, role):
        copier = oracle_factory(k_caches, v_caches, block_size, role)
        copier.format = format
        return copier
    return factory


@pytest.mark.parametrize("mine, theirs", [("mxint8", "mxfp8"), (None, "mxfp8"), ("mxfp8", None)])
@pytest.mark.parametrize("direct", [False, True])
def test_a_decode_worker_refuses_another_format_before_it_reserves(mine, theirs, direct):
    from iekv.serve.disaggregated import DecodeWorker, DirectSource

    worker = DecodeWorker(model(), engine_config(), copier_factory=tagged(mine))
    transfer = make_transfer(packed_of(theirs))
    transfer.first_block = 0
    if direct:
        copier = tagged(theirs)([torch.zeros(8, 2, 36)], [torch.zeros(8, 2, 36)], 4, "transfer")
        transfer.block_payloads, transfer.source = None, DirectSource(copier, [0, 1, 0], lambda: None)
    free = worker.engine.blocks.num_free
    with pytest.raises(ValueError, match=f"of {theirs or 'values'}, .* hold {mine or 'values'}"):
        worker.admit(transfer, max_new_tokens=4)
    scheduler = worker.engine.scheduler
    assert worker.engine.blocks.num_free == free
    assert not scheduler.waiting and not scheduler.running


def test_an_engine_tells_its_copiers_what_its_model_keeps():
    from iekv.engine.engine import Engine

    toy = model()
    assert Engine(toy, engine_config(), copier_factory=tagged(None)).make_copier().format is None
    toy.cache_format = "mxfp4"
    engine = Engine(toy, engine_config(offload_blocks=4, preemption="swap"),
                    copier_factory=tagged(None))
    assert {engine.make_copier().format, engine.copier.format, engine.swapper.format} == {"mxfp4"}
    plain = Engine(toy, engine_config(), copier_factory=oracle_factory)   # of no such knowledge
    assert not hasattr(plain.make_copier(), "format")


def test_what_a_copier_without_formats_moves_is_its_own_matter():
    from iekv.serve.disaggregated import DecodeWorker

    worker = DecodeWorker(model(), engine_config(), copier_factory=oracle_factory)
    worker._refuse_other_format(make_transfer(packed_of("mxfp8")))
    transfer = make_transfer(packed_of("mxfp8"))
    transfer.block_payloads = list(packed_of("mxfp8"))      # of a list each payload says, if it can
    DecodeWorker(model(), engine_config(),
                 copier_factory=tagged("mxint8"))._refuse_other_format(transfer)
