"""Token log probabilities, entropy and alternatives against the definition in 64 bits (GPU).

Tolerances, with u = 2^-24 and n the vocabulary: a difference x - m is rounded once and the
exponential is off by a few steps, so each term by |x - m| u + 4 u relative to itself, 2 R u
with R the range of the logits that matter (terms further than 104 below the largest are
zero); a sum of n terms adds at most (n / 256 + 64) u as it is split; the logarithm is off by
as much absolutely, plus 4 steps of its value; the logit and the difference are rounded once
each. Alternatives are whole numbers and must be equal.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def reference(logits, tokens, top):
    x = logits.double()
    # From the largest on: next to the types' lowest values x - lse would lose what counts.
    m = x.amax(1, keepdim=True)
    log_s = torch.log(torch.exp(x - m).sum(1, keepdim=True))
    lse = m + log_s
    lp = torch.where(torch.isneginf(x), float("-inf"), (x - m) - log_s)
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(1)
    picked = lp.gather(1, tokens[:, None])[:, 0]
    order = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :top]
    return picked, entropy, lp.gather(1, order), order, lse


def check(logits, tokens, top):
    from iekv.engine.logprobs import token_logprobs

    got = token_logprobs(logits, tokens, top=top)
    picked, entropy, tops, ids, lse = reference(logits, tokens, top)
    u, n = 2.0 ** -24, logits.shape[1]
    finite = logits.double().masked_fill(torch.isinf(logits), 0.0)
    spread = torch.minimum(finite.amax(1) - finite.amin(1), torch.tensor(104.0, device="cuda"))
    tol = u * (2 * spread + n / 256 + 80)
    size = torch.maximum(lse[:, 0].abs(), finite.abs().amax(1))
    assert torch.equal(got.top_ids, ids)

    def close(a, b, t):
        same = (a == b) | ((a.double() - b).abs() <= t)
        assert same.all(), ((a.double() - b).abs() / t).nan_to_num(0.0).max()

    close(got.logprobs, picked, tol + 4 * u * (size + picked.abs().nan_to_num(0, 0, 0)))
    # w / s is a mean of x - m weighted by p: off by the terms' errors times its size.
    mean = (finite.amax(1) - lse[:, 0]).abs() + entropy
    close(got.entropy, entropy, (tol + 8 * u) * (1 + mean + spread))
    close(got.top_logprobs, tops, (tol + 4 * u * size)[:, None] + 4 * u * tops.abs().nan_to_num(
        0, 0, 0))
    return got


def make(rows, vocab, dtype, seed, scale=2.5, masked=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, vocab), generator=gen, device="cuda") * scale
    if masked:
        x[torch.rand((rows, vocab), generator=gen, device="cuda") < masked] = float("-inf")
        x[:, vocab // 2] = 1.0                   # one token is left at least
    tokens = torch.randint(vocab, (rows,), generator=gen, device="cuda")
    return x.to(dtype), tokens


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows, vocab, top", [
    (1, 1, 1), (1, 2, 0), (3, 7, 7), (5, 63, 20), (2, 64, 64), (4, 65, 64), (64, 256, 5),
    (1, 1000, 1), (7, 4095, 33), (2, 4097, 64), (3, 50001, 20), (1, 128000, 20), (300, 999, 3),
    (33, 32000, 5), (1, 300007, 64)])
def test_sizes_and_types(gpu, dtype, rows, vocab, top):
    check(*make(rows, vocab, dtype, vocab + top), top)
    check(*make(rows, vocab, dtype, vocab + top + 1, masked=0.7), top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [100, 5000, 70001])
def test_ties_and_orders(gpu, dtype, vocab):
    """Equal logits go by index; rows that rise, fall, or hold one value everywhere."""
    at = torch.arange(vocab, device="cuda")
    rows = [torch.zeros(vocab, device="cuda"), at / vocab, -(at / vocab), (at % 7).float(),
            -(at % 5).float(), torch.where(at % 2 == 0, 0.0, -0.0),
            torch.where(at == vocab - 1, 5.0, 0.0), torch.where(at >= vocab - 70, 3.0, -1.0),
            torch.where(at % 64 == 63, (at / vocab), torch.full_like(at / vocab, -4.0))]
    x = torch.stack(rows).to(dtype)
    tokens = torch.tensor([0, vocab - 1, 1, 2, 3, 4, vocab - 1, vocab - 70, 63], device="cuda")
    check(x, tokens, 64)
    check(x, tokens, 1)


@pytest.mark.parametrize("vocab", [3, 1000, 20000])
def test_values_at_the_edges(gpu, vocab):
    from iekv.engine.logprobs import token_logprobs

    inf, nan = float("inf"), float("nan")
    for dtype in (F32, F16, BF16):
        x, tokens = make(6, vocab, dtype, 5)
        low = torch.finfo(dtype).min
        x[0] = -inf                              # nothing is left
        x[1] = low                               # the type's lowest value everywhere
        x[2, :-1] = -inf                         # one token is left
        x[3, 1] = nan
        x[4, 1] = inf
        x[5] = low
        x[5, 2] = torch.finfo(dtype).max
        tokens[:] = 2
        tokens[2] = vocab - 1
        got = token_logprobs(x, tokens, top=3)
        assert got.logprobs[0] == -inf and got.entropy[0] == 0
        assert got.top_ids[0].tolist() == [0, 1, 2] and (got.top_logprobs[0] == -inf).all()
        check(x[1:3], tokens[1:3], 3)
        assert got.logprobs[2] == 0 and got.entropy[2] == 0
        for row in (3, 4):
            assert got.logprobs[row].isnan() and got.entropy[row].isnan()
            assert got.top_logprobs[row].isnan().all() and got.top_ids[row, 0] == 1
        assert got.logprobs[5] == 0 and got.entropy[5] == 0
        for bad in (-1, vocab, 1 << 40):
            tokens[1] = bad
            got = token_logprobs(x, tokens)
            assert got.logprobs[1].isnan() and not got.entropy[1].isnan()


def test_strides_streams_graphs_and_repeats(gpu):
    from iekv.engine.logprobs import token_logprobs

    x, tokens = make(5, 30001, BF16, 6)
    want = check(x, tokens, 20)
    wide = torch.full((5, 30011), 9.0, dtype=BF16, device="cuda")
    wide[:, 3:30004] = x
    row = make(1, 501, F32, 7)
    check(row[0].expand(6, 501), torch.arange(6, device="cuda"), 4)
    for given in (wide[:, 3:30004], x.t().contiguous().t(),
                  wide.clone().flatten()[1:1 + 5 * 30001].view(5, 30001).copy_(x)):
        got = token_logprobs(given, tokens, top=20)
        assert torch.equal(got.top_ids, want.top_ids)
        check(given, tokens, 20)
    spread = torch.stack((tokens, tokens), 1)[:, 0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = token_logprobs(x, spread, top=20)
    torch.cuda.current_stream().wait_stream(side)
    for name in ("logprobs", "entropy", "top_logprobs", "top_ids"):
        assert torch.equal(getattr(got, name), getattr(want, name))
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = token_logprobs(static, tokens, top=20)
    for turn in range(3):
        fresh, _ = make(5, 30001, BF16, 8 + turn)
        static.copy_(fresh)
        graph.replay()
        eager = token_logprobs(fresh, tokens, top=20)
        torch.cuda.synchronize()
        for name in ("logprobs", "entropy", "top_logprobs", "top_ids"):
            assert torch.equal(getattr(got, name), getattr(eager, name))


def test_rows_past_32_bits(gpu):
    """More than 2^31 logits in one call."""
    rows, vocab = 17000, 128000
    x = torch.zeros((rows, vocab), dtype=BF16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(9)
    x[-3:] = torch.randn((3, vocab), generator=gen, device="cuda").to(BF16)
    tokens = torch.arange(rows, device="cuda") % vocab
    from iekv.engine.logprobs import token_logprobs

    got = token_logprobs(x, tokens, top=2)
    want = check(x[-3:].clone(), tokens[-3:], 2)
    assert torch.equal(got.top_ids[-3:], want.top_ids)
    assert torch.equal(got.logprobs[-3:], want.logprobs)
    assert (got.top_ids[:-3] == torch.tensor([0, 1], device="cuda")).all()


def test_refusals(gpu):
    from iekv.engine.logprobs import token_logprobs

    x, tokens = make(4, 100, F32, 10)
    for bad, given, top in ((x.double(), tokens, 0), (x.cpu(), tokens, 0), (x[0], tokens, 0),
                            (x, tokens[:3], 0), (x, tokens.int(), 0), (x, tokens.cpu(), 0),
                            (x, tokens, 65), (x, tokens, -1), (x[:, :4], tokens, 5)):
        with pytest.raises(ValueError):
            token_logprobs(bad, given, top=top)
    with pytest.raises(RuntimeError, match="vocab 0"):
        token_logprobs(x[:, :0], tokens)
    with pytest.raises(RuntimeError, match="backward"):
        token_logprobs(x.clone().requires_grad_(), tokens)
    got = token_logprobs(x[:0], tokens[:0], top=3)
    assert got.logprobs.shape == (0,) and got.top_ids.shape == (0, 3)
