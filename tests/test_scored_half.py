"""Half-precision weights of scored attention: keys far below the best one still count where there are many of them."""
import numpy as np
import pytest
import torch

from oracle.scored_ref import attend_ref
from test_scored_attn import DEV, HF

# A weight is rounded to half precision after a factor of 2^7: it keeps 11 bits or is off by 2^-25 of 2^7, 2^-32 of the first
# maximum's weight, and the weights' sum is at least that one.  So N keys lose N 2^-32 max |v| at most beside the usual bound.
LOST = 2.0 ** -32


def _case(n, below, rows, seed):
    """One request of n tokens, D = 64.  The first key leads all others by about `below` powers of two and has no value."""
    g = torch.Generator().manual_seed(seed)
    k = torch.randn((n, 1, 64), generator=g) * 0.02
    k[:, 0, 0] = 0.0
    k[0] = 0.0
    k[0, 0, 0] = 8.0
    q = torch.randn((rows, 2, 64), generator=g) * 0.1
    q[:, :, 0] = below * np.log(2.0)                                       # times the key's 8 and the scale 1/8
    v = 1.0 + 0.25 * torch.randn((n, 1, 64), generator=g)
    v[0] = 0.0
    return q.to(HF), k.to(HF), v.to(HF)


@pytest.mark.parametrize("below", [12.0, 20.0, 25.3])
def test_what_half_precision_loses(below):
    """The bound by arithmetic alone: weights rounded after the factor stay within it, without the factor they do not."""
    n = 40000
    q, k, v = _case(n, below, 1, 1)
    x = (k[:, 0].double() @ q[0, 0].double()) / 8
    w = torch.exp(x - x.max())
    want = (w / w.sum()) @ v[:, 0].double()
    lift = lambda f: ((w * f).to(HF).double() @ v[:, 0].double()) / (w.sum() * f)  # noqa: E731
    tol = torch.finfo(HF).eps / 2 * ((w / w.sum()) @ v[:, 0].double().abs()) + n * LOST * float(v.abs().max())
    assert bool(((lift(128.0) - want).abs() <= tol).all())
    if below > 24:
        assert bool(((lift(1.0) - want).abs() > 20 * tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("below", [12.0, 20.0, 25.3])
@pytest.mark.parametrize("B", [1, 300], ids=["split", "whole"])
@pytest.mark.parametrize("rows", [1, 9], ids=["single", "extend"])
def test_many_small_weights(rows, B, below):
    """One request whose keys are cut into parts, and 300 of the same tokens, each walked whole: there all keys meet the best one."""
    from mi355_attn import ops
    n = 40000
    q, k, v = _case(n, below, rows, 2)
    form = {} if rows == 1 else dict(prefix_lens=torch.full((B,), n - rows, device=DEV), max_extend_len=rows,
                                     cu_q=torch.arange(0, B * rows + 1, rows, dtype=torch.int32, device=DEV))
    for kw in (dict(), dict(softcap=1000.0)):
        got = ops.scored_attn(q.reshape(rows, -1).repeat(B, 1).to(DEV), k.to(DEV), v.to(DEV), torch.arange(n // 16, dtype=torch.int32, device=DEV)[None],
                              torch.zeros(B, dtype=torch.int64, device=DEV), torch.full((B,), n, device=DEV), 16, 2, n, **form, **kw)
        keys = [list(range(n - rows + 1 + j)) for j in range(rows)]
        want, tol = attend_ref(q, k, v, range(n), [(s, s, len(s) - 1) for s in keys], HF, 0.125, **kw)
        # (a result below 2^-14 is itself rounded in steps of 2^-24)
        tol = tol + n * LOST * float(v.abs().max()) + 2.0 ** -25
        off = (got.double().cpu().view(B, *want.shape) - want).abs() - tol
        assert float(off.max()) <= 0
