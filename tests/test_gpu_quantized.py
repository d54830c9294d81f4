"""Microscaled caches: rows quantised as they are written, and read back (GPU).

The format leaves nothing open: the bytes that are written have to be those of the definition
(the sign of a zero apart), and the values that are read those that the bytes stand for, rounded
once to the type asked for.
"""
from __future__ import annotations

import pytest
import torch

from quantized_reference import FORMATS, decode, encode, same_records

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def make_pool(blocks, bs, heads, dim, format, layers=1, fill=None):
    from iekv.engine.quantized import QuantizedPool, allocate_quantized_pool

    k, v = allocate_quantized_pool(blocks, bs, layers, heads, dim, format=format)
    if fill is not None:
        for t in k + v:
            t.fill_(fill)
    return QuantizedPool(k, v, bs, format), k, v


def rows_of(shape, dtype, seed, scale=1.0):
    """Values over many magnitudes: whole rows, and single channels, some of them zero."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(s, generator=gen, device="cuda")

    x = normal(*shape) * torch.exp2(normal(*shape[:-1], 1) * 4).mul(scale)
    x *= torch.exp2(normal(*shape[-2:]))
    x[normal(*shape) > 1.5] = 0
    return x.to(dtype)


def same(got, want):
    """Equal values, NaN where NaN is."""
    return torch.equal(torch.nan_to_num(got, nan=12345.0), torch.nan_to_num(want, nan=12345.0))


SHAPES = [(1, 8, 4), (2, 16, 16), (4, 32, 16), (3, 40, 8), (5, 80, 16), (1, 72, 1), (2, 64, 256),
          (8, 128, 16), (3, 104, 3), (16, 96, 16), (1, 128, 16), (7, 120, 5)]


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads, dim, bs", SHAPES)
@pytest.mark.parametrize("n", [1, 37])
def test_rows_are_held_and_read_back_by_the_definition(gpu, format, dtype, heads, dim, bs, n):
    from iekv.engine.slots import gather_rows, gather_rows_arrays, write_slots, write_slots_layers

    layers, blocks = 2, -(-n // bs) + 2
    pool, k, v = make_pool(blocks, bs, heads, dim, format, layers, fill=0xa5)
    rows = rows_of((2, layers, n, heads, dim), dtype, n + dim)
    gen = torch.Generator().manual_seed(n)
    table = torch.randperm(blocks, generator=gen)[:-(-n // bs)].tolist()
    slots = [table[j // bs] * bs + j % bs for j in range(n)]
    write_slots_layers(pool, rows[0], rows[1], torch.tensor(slots, device=gpu))
    want = encode(rows, format)
    for l in range(layers):
        for o, cache in ((0, k), (1, v)):
            assert same_records(cache[l][slots], want[o, l], format)
            rest = torch.ones(blocks * bs, dtype=torch.bool)
            rest[slots] = False
            assert (cache[l].cpu()[rest] == 0xa5).all()
    values = decode(want, format)
    for out in TYPES:
        got = gather_rows_arrays(pool, table, n, dtype=out)
        assert got.dtype == out and same(got.cpu(), values.flatten(0, 1).to(F32).to(out))
    # One layer alone, from host slots, and one array of it.
    write_slots(pool, 1, rows[0, 0], rows[1, 0], slots)
    assert same_records(k[1][slots], want[0, 0], format)
    assert same_records(k[0][slots], want[0, 0], format)
    assert same(gather_rows(pool, 3, table, n).cpu(), values[1, 0].to(BF16))


def every(dtype):
    """Every number of a 16-bit type; of float32 those with few bits, of each exponent."""
    if dtype == F32:
        part = torch.cat((torch.arange(0, 1 << 23, 1 << 16), torch.tensor([1, 0x600001, 0x400001,
                                                                            0x7e0001, 0x7fffff])))
        bits = (torch.arange(256)[:, None] << 23 | part).reshape(-1)
        return torch.cat((bits, bits - (1 << 31))).to(torch.int32).view(F32)
    return torch.arange(-(1 << 15), 1 << 15).to(torch.int16).view(dtype)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_every_number(gpu, format, dtype):
    """As the largest of its group, and under largest ones of 1 to 2^9 times its size."""
    from iekv.engine.slots import gather_rows, write_slots

    x = every(dtype)
    dim, bs = 32, 64
    n = len(x)
    rows = torch.zeros((n, 4, dim), dtype=dtype)
    rows[:, :, 5] = x[:, None]
    power = torch.tensor([0, 3, 6, 9])
    largest = (x[:, None].abs().double() * torch.exp2(power.double()) * 1.25).to(dtype)
    rows[:, 1:, 17] = -largest[:, 1:]
    blocks = -(-n // bs)
    pool, k, _ = make_pool(blocks, bs, 4, dim, format)
    on = rows.to(gpu)
    slots = torch.arange(n, device=gpu)
    write_slots(pool, 0, on, on, slots)
    want = encode(rows, format)
    assert same_records(k[0][:n], want, format)
    values = decode(want, format)
    for out in TYPES:
        got = gather_rows(pool, 0, list(range(blocks)), n, dtype=out)
        assert same(got.cpu(), values.to(F32).to(out))


@pytest.mark.parametrize("format", FORMATS)
def test_every_record_is_read(gpu, format):
    """Every code with every exponent, whoever wrote them."""
    from iekv.engine.slots import gather_rows

    pool, k, v = make_pool(16, 16, 256, 16, format)
    codes = k[0].shape[2] - 4
    records = torch.zeros((256, 256, codes + 4), dtype=torch.uint8)
    records[:, :, :codes] = torch.arange(256)[None, :, None]
    records[:, :, codes] = torch.arange(256)[:, None]
    records[:, :, codes + 1:] = 77                 # of no group
    k[0].copy_(records)
    values = decode(records, format)
    if format == "mxint8":                         # no such exponent is written
        values[0] = 0
        finite = torch.isfinite(values) | (records[:, :, codes, None] != 255)
        values = torch.where(finite, values, float("nan"))
    for out in TYPES:
        got = gather_rows(pool, 0, list(range(16)), 256, dtype=out).cpu()
        want = values.to(F32).to(out)
        if format == "mxint8":                     # codes of a group with 255 are zeros
            got, want = got[:255], want[:255]
        assert same(got, want)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_groups_with_nan_or_infinity(gpu, format, dtype):
    from iekv.engine.slots import gather_rows, write_slots

    pool, k, v = make_pool(1, 8, 2, 80, format, fill=1)
    rows = rows_of((3, 2, 80), dtype, 4)
    rows[0, 0, 7] = float("nan")
    rows[0, 1, 40] = float("inf")
    rows[1, 1, 79] = -float("inf")
    write_slots(pool, 0, rows, rows, [2, 0, 7])
    assert same_records(v[0][[2, 0, 7]], encode(rows, format), format)
    got = gather_rows(pool, 0, [0], 8, dtype=F32)[[2, 0, 7]].cpu()
    nan = torch.isnan(got)
    want = torch.zeros_like(nan)
    want[0, 0, :32] = want[0, 1, 32:64] = want[1, 1, 64:] = True
    assert torch.equal(nan, want)


@pytest.mark.parametrize("format", FORMATS)
def test_strided_rows(gpu, format):
    """K and V as slices of one projection, heads far apart, dimensions that are not contiguous,
    layers in another order, and one row for all tokens."""
    from iekv.engine.slots import write_slots, write_slots_layers

    pool, k, v = make_pool(4, 16, 3, 40, format, layers=3)
    n = 21
    slots = torch.arange(n, device=gpu) * 3 % 64
    qkv = rows_of((n, 9, 40), BF16, 3)
    write_slots(pool, 1, qkv[:, 3:6], qkv[:, 6:], slots)
    assert same_records(k[1][slots], encode(qkv[:, 3:6], format), format)
    assert same_records(v[1][slots], encode(qkv[:, 6:], format), format)
    x = rows_of((3, n, 3, 40), F32, 5)
    write_slots(pool, 0, x.permute(3, 1, 2, 0).contiguous().permute(1, 2, 0, 3)[..., 0],
                x[2].transpose(0, 1).contiguous().transpose(0, 1), slots)
    assert same_records(k[0][slots], encode(x[0], format), format)
    assert same_records(v[0][slots], encode(x[2], format), format)
    write_slots_layers(pool, x.flip(0), x.transpose(0, 1).contiguous().transpose(0, 1), slots)
    for l in range(3):
        assert same_records(k[l][slots], encode(x[2 - l], format), format)
        assert same_records(v[l][slots], encode(x[l], format), format)
    one = x[0, :1].expand(n, 3, 40)
    write_slots(pool, 2, one, one, slots)
    assert same_records(k[2][slots], encode(one, format), format)
    # A conjugate's imaginary part is a negated view.
    z = torch.complex(x[0], x[1])
    write_slots(pool, 2, z.conj().imag, x[0], slots)
    assert same_records(k[2][slots], encode(-x[1], format), format)


def test_arrays_at_any_distance(gpu):
    """A pool of separate tensors, at odd addresses and in no order."""
    from iekv.engine.quantized import QuantizedPool, record_bytes
    from iekv.engine.slots import gather_rows_arrays, write_slots_layers

    format, heads, dim, bs, blocks, layers = "mxfp4", 3, 24, 4, 5, 5
    size = blocks * bs * heads * record_bytes(format, dim)
    flat = torch.full((40 * size,), 0x3c, dtype=torch.uint8, device=gpu)
    at = [17 + 2 * size * i + 3 * (i % 3) for i in (7, 3, 12, 1, 9, 10, 2, 15, 5, 18)]
    arrays = [flat[a:a + size].view(blocks * bs, heads, -1) for a in at]
    pool = QuantizedPool(arrays[:layers], arrays[layers:], bs, format)
    rows = rows_of((2, layers, 9, heads, dim), F16, 8)
    table = [4, 0, 2]
    slots = torch.tensor([table[j // bs] * bs + j % bs for j in range(9)], device=gpu)
    write_slots_layers(pool, rows[0], rows[1], slots)
    want = encode(rows, format).flatten(0, 1)
    for a, w in zip(arrays, want):
        assert same_records(a[slots], w, format)
    got = gather_rows_arrays(pool, table, 9, first_array=2, n_arrays=7, dtype=F32)
    assert same(got.cpu(), decode(want, format).to(F32)[2:9])
    for a in arrays:
        a.fill_(0x3c)
    assert (flat == 0x3c).all()


@pytest.mark.parametrize("format", FORMATS)
def test_device_slots_and_blocks_outside_the_pool(gpu, format):
    from iekv.engine.slots import gather_rows, write_slots

    pool, k, v = make_pool(3, 8, 2, 48, format, fill=0x11)
    rows = rows_of((6, 2, 48), BF16, 1)
    slots = torch.tensor([23, 24, -1, 0, 1 << 40, -(1 << 62)], device=gpu)
    write_slots(pool, 0, rows, rows, slots)
    want = torch.full_like(k[0], 0x11).cpu()
    want[[23, 0]] = encode(rows[[0, 3]], format)
    assert same_records(k[0], want, format) and same_records(v[0], want, format)
    out = gather_rows(pool, 0, torch.tensor([2, 3, 0], device=gpu), 24, dtype=F32)
    assert same(out[16:].cpu(), decode(k[0][:8], format).to(F32))
    assert same(out[:8].cpu(), decode(k[0][16:], format).to(F32))


def test_blocks_past_32_bits_are_outside_the_pool(gpu):
    """As entries of a table of 64 bits, of which a kernel takes 32."""
    pool, _, _ = make_pool(3, 8, 2, 48, "mxfp8")
    for wide in (1 << 32, (1 << 32) + 1, -(1 << 32), (1 << 62) + 2, 3, -1):
        table, _ = pool._table(torch.tensor([2, wide, 0], device=gpu), 24)
        first, bad, last = table.tolist()
        assert (first, last) == (2, 0) and not 0 <= bad < 3


@pytest.mark.parametrize("format", FORMATS)
def test_nothing_to_do(gpu, format):
    from iekv.engine.slots import gather_rows, gather_rows_arrays, write_slots, write_slots_layers

    pool, k, v = make_pool(2, 8, 2, 32, format, layers=2, fill=9)
    empty = torch.empty((0, 2, 32), device=gpu)
    write_slots(pool, 0, empty, empty, [])
    write_slots(pool, 0, empty, empty, torch.empty(0, dtype=torch.int64, device=gpu))
    write_slots_layers(pool, empty[None], empty[None], [])
    assert gather_rows(pool, 1, [], 0, dtype=F16).shape == (0, 2, 32)
    assert gather_rows_arrays(pool, [1], 0).shape == (4, 0, 2, 32)
    assert all((t == 9).all() for t in k + v)


@pytest.mark.parametrize("n", [1, 127, 128, 129, 256, 257, 600, 1500])
def test_lists_of_any_length(gpu, n):
    """Slots and tables on the host, carried in one launch, in two, and uploaded."""
    from iekv.engine.slots import gather_rows, gather_rows_arrays, write_slots, write_slots_layers

    format, bs = "mxint8", 1
    pool, k, v = make_pool(n + 40, bs, 2, 24, format, layers=2)
    gen = torch.Generator().manual_seed(n)
    slots = torch.randperm(n + 40, generator=gen)[:n]
    rows = rows_of((2, 2, n, 2, 24), F16, n)
    write_slots_layers(pool, rows[0], rows[1], slots.tolist())
    want = encode(rows, format)
    for given in (slots.tolist(), slots, slots.numpy(), slots.to(gpu), slots.to(gpu).int()):
        got = gather_rows_arrays(pool, given, n, dtype=F32)
        assert same(got.cpu(), decode(want, format).to(F32).flatten(0, 1))
    for given in (slots, slots.numpy().astype("int32"), tuple(slots.tolist()), slots.to(gpu).int()):
        k[1].zero_()
        write_slots(pool, 1, rows[0, 1], rows[1, 1], given)
        assert same_records(k[1][slots], want[0, 1], format)
    # Of blocks of several rows, of which the context's last holds some.
    wide, *_ = make_pool(n, 3, 2, 24, format)
    write_slots(wide, 0, rows[0, 0], rows[1, 0], list(range(3, 3 + n)) if n > 1 else [0])
    blocks = list(range(1, -(-n // 3) + 1)) if n > 1 else [0]
    got = gather_rows(wide, 1, blocks, n, dtype=F32)
    assert same(got.cpu(), decode(want, format).to(F32)[1, 0])


def test_offsets_past_32_bits(gpu):
    """Rows, caches and values behind the first 4 GiB."""
    from iekv.engine.slots import gather_rows, write_slots

    format, heads, dim, bs = "mxfp8", 8, 128, 16
    blocks = 300_000                                    # 5 GB an array
    pool, k, v = make_pool(blocks, bs, heads, dim, format)
    assert k[0].numel() > 1 << 32
    rows = rows_of((40, heads, dim), BF16, 2)
    slots = torch.arange(blocks * bs - 40, blocks * bs, device=gpu)
    write_slots(pool, 0, rows, rows, slots)
    assert same_records(v[0][-40:], encode(rows, format), format)
    assert not k[0][:-40].view(-1).view(torch.int32).any()
    # 2.4 million rows of 2 KiB, the last ones of them what was written.
    n = 2_400_000
    out = gather_rows(pool, 0, list(range(blocks - n // bs, blocks)), n)
    assert out.numel() * 2 > 1 << 32
    assert same(out[-40:].cpu(), decode(encode(rows, format), format).to(BF16))
    assert not out[:-40].any()


@pytest.mark.parametrize("format", FORMATS)
def test_streams_and_graphs(gpu, format):
    """A captured write and read, replayed on new rows, slots and tables, with eager calls
    between, on another stream too."""
    from iekv.engine.slots import gather_rows, write_slots

    pool, k, v = make_pool(8, 16, 2, 64, format)
    rows = rows_of((10, 2, 64), BF16, 1)
    slots = torch.arange(10, device=gpu)
    table = torch.tensor([0, 1], dtype=torch.int32, device=gpu)
    long, *_ = make_pool(600, 1, 2, 64, format)
    many = rows_of((300, 2, 64), BF16, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        write_slots(pool, 0, rows, rows, slots)
        gather_rows(pool, 0, table, 20)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        write_slots(pool, 0, rows, rows, slots)
        out = gather_rows(pool, 0, table, 20)
        listed = gather_rows(pool, 0, [3, 1], 20)     # a short list travels with its launch
        with pytest.raises(RuntimeError, match="capture"):
            write_slots(long, 0, many, many, list(range(300)))
        with pytest.raises(RuntimeError, match="capture"):
            gather_rows(long, 0, list(range(600)), 600)
    for seed in range(4):
        rows.copy_(rows_of((10, 2, 64), BF16, seed + 9))
        slots.copy_(torch.randperm(128, generator=torch.Generator().manual_seed(seed))[:10])
        table.copy_(torch.tensor([slots[0] // 16, slots[1] // 16]))
        graph.replay()
        eager = gather_rows(pool, 0, table, 20)
        torch.cuda.synchronize()
        assert same_records(k[0][slots], encode(rows, format), format)
        assert same(out, eager) and same(listed, gather_rows(pool, 0, [3, 1], 20))


def test_refusals(gpu):
    from iekv.engine.pools import KVPool
    from iekv.engine.quantized import QuantizedPool, allocate_quantized_pool
    from iekv.engine.slots import gather_rows, gather_rows_arrays, write_slots, write_slots_layers

    pool, k, v = make_pool(4, 8, 2, 32, "mxfp8", layers=2, fill=7)
    rows = rows_of((3, 2, 32), BF16, 1)
    slots = torch.arange(3, device=gpu)
    bad = [
        (ValueError, "slots for", lambda: write_slots(pool, 0, rows, rows, [1, 2])),
        (ValueError, "do not fit", lambda: write_slots(pool, 0, rows[..., :24], rows[..., :24], slots)),
        (ValueError, "must both be", lambda: write_slots(pool, 0, rows, rows[:, :1], slots)),
        (ValueError, "do not fit", lambda: write_slots(pool, 0, rows[:, :1], rows[:, :1], slots)),
        (ValueError, "must both be", lambda: write_slots(pool, 0, rows, rows[:2], slots)),
        (ValueError, "must both be", lambda: write_slots_layers(pool, rows, rows, slots)),
        (ValueError, "slots of shape", lambda: write_slots(pool, 0, rows, rows, slots[:2])),
        (ValueError, "slots of shape",
         lambda: write_slots(pool, 0, rows, rows, slots[:, None].repeat(1, 2))),
        (ValueError, "6 slots",
         lambda: write_slots(pool, 0, rows, rows, torch.arange(6).view(3, 2))),
        (ValueError, "table of 4", lambda: gather_rows(pool, 0, [[1, 2], [3, 0]], 16)),
        (TypeError, "one dimension", lambda: gather_rows(pool, 0, slots[:, None], 16)),
        (TypeError, "integer", lambda: gather_rows(pool, 0, [1], 8.0)),
        (IndexError, "layers 2..2", lambda: write_slots(pool, 2, rows, rows, slots)),
        (IndexError, "layers -1..-1", lambda: write_slots(pool, -1, rows, rows, slots)),
        (IndexError, "layers 1..2",
         lambda: write_slots_layers(pool, rows[None].repeat(2, 1, 1, 1),
                                    rows[None].repeat(2, 1, 1, 1), slots, first_layer=1)),
        (IndexError, "slot 32", lambda: write_slots(pool, 0, rows, rows, [1, 32, 2])),
        (IndexError, "slot -1", lambda: write_slots(pool, 0, rows, rows, [1, -1, 2])),
        (ValueError, "distinct", lambda: write_slots(pool, 0, rows, rows, [1, 3, 1])),
        (TypeError, "integers", lambda: write_slots(pool, 0, rows, rows, [1.0, 2.0, 3.0])),
        (TypeError, "integers", lambda: write_slots(pool, 0, rows, rows, slots.float())),
        (ValueError, "float64", lambda: write_slots(pool, 0, rows.double(), rows.double(), slots)),
        (ValueError, "V rows of", lambda: write_slots(pool, 0, rows, rows.float(), slots)),
        (ValueError, "on cpu", lambda: write_slots(pool, 0, rows.cpu(), rows, slots)),
        (RuntimeError, "no backward",
         lambda: write_slots(pool, 0, rows.clone().requires_grad_(), rows, slots)),
        (IndexError, "needs 3 blocks", lambda: gather_rows(pool, 0, [1, 2], 17)),
        (IndexError, "block id 4", lambda: gather_rows(pool, 0, [1, 4], 16)),
        (IndexError, "arrays 4..4", lambda: gather_rows(pool, 4, [1], 8)),
        (IndexError, "arrays", lambda: gather_rows_arrays(pool, [1], 8, 3, 2)),
        (ValueError, "context", lambda: gather_rows(pool, 0, [1], -1)),
        (ValueError, "float64", lambda: gather_rows(pool, 0, [1], 8, dtype=torch.float64)),
        (TypeError, "block table", lambda: gather_rows(pool, 0, slots.float(), 8)),
        (ValueError, "no format", lambda: QuantizedPool(k, v, 8, "mxfp6")),
        (ValueError, "none of mxfp4", lambda: QuantizedPool(
            [k[0][..., :5].contiguous()], [v[0][..., :5].contiguous()], 8, "mxfp4")),
        (ValueError, "uint8", lambda: QuantizedPool(
            [k[0].view(torch.int8)], [v[0].view(torch.int8)], 8, "mxfp8")),
        (ValueError, "head_dim 136", lambda: allocate_quantized_pool(
            4, 8, 1, 2, 136, format="mxfp8")),
        (ValueError, "head_dim 12", lambda: allocate_quantized_pool(
            4, 8, 1, 2, 12, format="mxint8")),
        (ValueError, "not as", lambda: gather_rows(KVPool(k, v, 8), 0, [1], 8, dtype=BF16)),
    ]
    for kind, said, call in bad:
        with pytest.raises(kind, match=said):
            call()
    torch.cuda.synchronize()
    assert all((t == 7).all() for t in k + v)
    # The records themselves, as bytes.
    raw = gather_rows(KVPool(k, v, 8), 0, [1], 8)
    assert raw.dtype == torch.uint8 and raw.shape == (8, 2, 36)


@pytest.mark.parametrize("kind", ["int64", "int32", "uint8", "int8"])
def test_layers_are_whole_numbers_of_any_kind(gpu, kind):
    """NumPy's among them, as of other pools: 40 of 8 bits times 8 would be past their end."""
    import numpy as np

    from iekv.engine.slots import gather_rows, gather_rows_arrays, write_slots, write_slots_layers

    kind = np.dtype(kind).type
    pool, _, _ = make_pool(2, 4, 1, 32, "mxint8", layers=41)
    k, v = (rows_of((2, 3, 1, 32), F32, seed) for seed in (91, 92))
    write_slots(pool, kind(40), k[0], v[0], [1, 2, 3])
    write_slots_layers(pool, k, v, [4, 5, 6], first_layer=kind(38))
    for layer, slots, x in ((40, [1, 2, 3], k[0]), (38, [4, 5, 6], k[0]), (39, [4, 5, 6], k[1])):
        got = gather_rows_arrays(pool, [0, 1], kind(8), first_array=kind(layer), n_arrays=kind(2),
                                 dtype=F32)
        assert torch.equal(got[0, slots], decode(encode(x, "mxint8"), "mxint8").float().cuda())
        assert torch.equal(gather_rows(pool, kind(layer), [0, 1], 8, dtype=F32), got[0])
    got = gather_rows(pool, kind(81), [0, 1], 8, dtype=F32)           # V of the last layer
    assert torch.equal(got[1:4], decode(encode(v[0], "mxint8"), "mxint8").float().cuda())
    for first, n in ((81, 100), (82, 1), (40, 0)):                   # 181 of 8 bits is below 0
        with pytest.raises(IndexError, match="out of range for 82 arrays"):
            gather_rows_arrays(pool, [0, 1], 8, first_array=kind(first), n_arrays=kind(n))
    with pytest.raises(IndexError, match="out of range for 41 layers"):
        write_slots_layers(pool, k, v, [4, 5, 6], first_layer=kind(40))
    with pytest.raises(TypeError):
        write_slots(pool, 1.0, k[0], v[0], [1, 2, 3])
