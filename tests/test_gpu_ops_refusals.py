"""What the operators refuse of real tensors (GPU)."""
from __future__ import annotations

import pytest
import torch

from test_gpu_attention import BF16, F32, make_pool, queries_of

pytestmark = pytest.mark.gpu


def test_tangents_are_refused(gpu):
    """A dual tensor requires no gradient: its tangent would be dropped in silence."""
    from torch.autograd import forward_ad

    from iekv.engine.attention import AttentionPlan, attend
    from iekv.engine.logprobs import token_logprobs

    pool, k, v = make_pool(4, 16, 2, 64, BF16, 1)
    plan = AttentionPlan(pool, [[1, 2]], [20], [1], 8)
    q = queries_of(1, 8, 64, BF16, 2)
    logits = torch.randn((3, 50), dtype=F32, device="cuda")
    tokens = torch.arange(3, device="cuda")
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward mode"):
            attend(plan, 0, forward_ad.make_dual(q, torch.ones_like(q)))
        with pytest.raises(RuntimeError, match="forward mode"):
            token_logprobs(forward_ad.make_dual(logits, torch.ones_like(logits)), tokens)
        attend(plan, 0, q)
        token_logprobs(logits, tokens)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: attend(plan, 0, x), (q,), (torch.ones_like(q),))


@pytest.mark.parametrize("vocab, top", [(5, 2), (3, 0)])
def test_more_rows_than_a_launch_has_workgroups(gpu, vocab, top):
    """2^24 and some rows: the last ones, of a second launch, and the first are scored alike."""
    from iekv.engine.logprobs import token_logprobs

    rows = (1 << 24) + 1000
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((2000, vocab), generator=gen, device="cuda").to(BF16)
    logits = x.repeat(rows // 2000 + 1, 1)[:rows]
    tokens = (torch.arange(rows, device="cuda") % 2000) % vocab
    got = token_logprobs(logits, tokens, top=top)
    want = token_logprobs(x, tokens[:2000].clone(), top=top)
    index = torch.arange(rows, device="cuda") % 2000
    for name in ("logprobs", "entropy", "top_logprobs", "top_ids"):
        assert torch.equal(getattr(got, name), getattr(want, name)[index])
    lp = torch.log_softmax(x.double(), 1)
    assert ((want.logprobs - lp.gather(1, tokens[:2000, None])[:, 0]).abs() < 1e-6).all()
