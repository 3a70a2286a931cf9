"""Attention over the paged cache where one sequence of a batch is not what the call says: the others get their results."""
import math

import pytest
import torch

from tests import attnref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _ops(built_libs):
    import distserve_b200

    distserve_b200.load_ops()


# One sequence has more rows than max_rows says; the others are cut into parts, so the grid is sized for less work than a
# count of its rows would suggest.
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("others,most", [([1] * 24, 1), ([1] * 40, 1), ([70] * 5 + [1] * 4, 70), ([70] * 34, 70)], ids=["steps", "many", "chunks", "manychunks"])
def test_a_sequence_of_too_many_rows_leaves_the_others_alone(others, most, e4m3):
    too_many, kv_heads, dim = 500, {24: 12, 40: 4}.get(len(others), 2), 64
    lengths = 3600 if most == 1 else 2000
    p = R.make_paged(41, [too_many] + others, [0] + [lengths - n - 20 * i for i, n in enumerate(others)], kv_heads, dim, 16, "fp16", e4m3, layers=1, layer=0)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(too_many + sum(others), kv_heads, dim, generator=g).half()
    d = p.to("cuda")
    junk = torch.full((64 << 20,), math.nan, device="cuda")              # what a workspace may hold before the call
    del junk
    out = torch.full_like(q, 7.0, device="cuda")
    torch.ops.kv_attention_ops.paged(q.cuda(), d.k_cache, d.v_cache, 0, d.tables, d.lens, d.starts, most, 0.125, out)
    out = out.cpu()
    assert torch.isnan(out[:too_many]).all()
    starts = p.starts.tolist()
    for i in range(1, len(others) + 1):
        a, b = starts[i], starts[i + 1]
        want = R.attend(q[a:b], R.rows_of(p, p.k_cache, i), R.rows_of(p, p.v_cache, i), 0.125, "fp16", e4m3)
        R.assert_close(out[a:b], want, f"sequence {i}")
