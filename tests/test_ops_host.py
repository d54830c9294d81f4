"""What the operators' library decides on the host (CPU)."""
from __future__ import annotations

import pytest

from test_attention_plan import make, ops  # noqa: F401  (the library, and a plan of two sequences)

INVALID = -1


@pytest.mark.parametrize("q, out, strides", [
    (1 << 20, (1 << 20) + 64, (512, 64)),          # some bytes further on
    ((1 << 20) + 16, 1 << 20, (512, 64)),
    (1 << 20, (1 << 20) + 6 * 1024 - 2, (512, 64)),    # the last element alone
    (1 << 20, 1 << 20, (64, 384)),                 # the same bytes in another order
    (1 << 20, 1 << 20, (1024, 64)),                # rows that lie further apart
    (1 << 20, 1 << 20, (0, 64)),                   # one row for all
    (1 << 20, (1 << 20) - 2048, (-512, 64)),       # rows that go back
])
def test_outputs_over_other_queries_are_refused(ops, q, out, strides):  # noqa: F811
    rc, plan, _ = make(ops)                        # 6 tokens of 8 heads of 64, 16 bits
    assert rc == 0
    assert ops.iekv_attend(plan, 64, 128, 192, q, *strides, 1.0, out, None, 0, None) == INVALID
    assert "overlaps" in ops.iekv_ops_last_error().decode()
    ops.iekv_attention_plan_destroy(plan)
