"""Scored attention at its limits, held to values: scores in the thousands, offsets and lengths that contradict each other."""
import pytest
import torch

from test_scored_attn import BF, DEV, Case, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("amp", [300.0, 3000.0])
@pytest.mark.parametrize("ext", [1, 7, 40], ids=["single", "few", "wide"])
def test_huge_scores_are_right(ext, amp):
    """Softmaxes of almost one key: the bound's score error (a sum of 64 products of thousands in 32 bits) is a fraction of one, so it
    still tells a right choice from a wrong one."""
    c = Case(80, BF, (2, 1, 64), 16, [60 - ext, 200], [ext, ext], amp=amp)
    want, tol = c.want()
    assert float((tol / c.v.nan_to_num().double().abs().max()).median()) < 0.25
    check(c.run(decode=ext == 1), want, tol)
    check(c.run(decode=ext == 1, softcap=50.0), *c.want(softcap=50.0))


CONTRADICTIONS = [  # cu_q, prefix lengths, lengths, rows that are still a request's own and in order, rows of no request
    ([0, 4, 100], [30, 5], [34, 9], [0, 1, 2, 3, 4, 5, 6, 7], []),
    ([0, 4, 8], [30, 2 ** 40], [34, 9], [0, 1, 2, 3], []),
    ([0, 4, 8], [30, 5], [34, -3], [0, 1, 2, 3], []),
    ([0, 4, 4], [30, 5], [34, 5], [0, 1, 2, 3], [4, 5, 6, 7]),
    ([0, 0, 0], [1, 1], [1, 1], [], [0, 1, 2, 3, 4, 5, 6, 7]),
    ([4, 0, 8], [30, 5], [34, 9], [], []),
    ([0, 4, 8], [-7, 2 ** 40], [2 ** 40, -3], [], []),
]


@pytest.mark.parametrize("cu,pre,lens,right,nobody", CONTRADICTIONS)
@pytest.mark.parametrize("hint", [40, 4000], ids=["whole", "parts"])
def test_contradictory_batches(cu, pre, lens, right, nobody, hint):
    """Requests that are in order are right beside others that are not, rows of no request keep what they held, and finite pools give
    finite rows."""
    from mi355_attn import ops
    c = Case(81, BF, (4, 2, 64), 16, [30, 5], [4, 4])
    want, tol = c.want()
    table = torch.where(c.table == 2 ** 31 - 1, 0, c.table)                # (columns past a request: some page of the pool)
    k, v = c.pool(c.k.nan_to_num()), c.pool(c.v.nan_to_num())
    out = torch.full((8, 256), 7.0, dtype=BF, device=DEV)
    ops.scored_attn(c.q.reshape(8, -1).to(DEV), k, v, table.to(DEV), c.rows.to(DEV), torch.tensor(lens, device=DEV), 16, 4, hint,
                    prefix_lens=torch.tensor(pre, device=DEV), cu_q=torch.tensor(cu, dtype=torch.int32, device=DEV), max_extend_len=8, out=out)
    got = out.view(8, 4, 64)
    assert bool(torch.isfinite(got).all())
    assert bool((got[nobody] == 7.0).all())
    if right:
        check(got[right], want[right], tol[right])
