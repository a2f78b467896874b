"""Draft trees on the GPU: metadata against whole-number rules, attention against the definition in 64 bits."""
import random

import numpy as np
import pytest
import torch

from oracle.scored_ref import ancestors_ref, attend_ref
from test_scored_attn import BF, DEV, HF, Case, check, slopes_of

pytestmark = pytest.mark.gpu


def trees(seed, sizes, bad=False):
    rng = random.Random(seed)
    out = []
    for n in sizes:
        p = [rng.randint(max(-1, j - 8), j - 1) for j in range(n)]
        if bad and n > 3:
            p[2], p[3] = 2, 9999                                          # itself and a node that is not there: roots
        out.append(p)
    return out


def prepare(c, parents, table=None, **kw):
    from mi355_attn import ops
    flat = torch.tensor([x for p in parents for x in p], dtype=torch.int32, device=DEV)
    return ops.tree_prepare(c.table.to(DEV) if table is None else table, c.rows.to(DEV), torch.tensor(c.pre, dtype=torch.int64, device=DEV), flat,
                            torch.tensor(c.cu, dtype=torch.int32, device=DEV), c.ps, max(c.ext), **kw)


def attn(c, plan, **kw):
    from mi355_attn import ops
    return ops.tree_attn(c.q.reshape(c.T, -1).to(DEV), c.pool(c.k), c.pool(c.v), c.table.to(DEV), c.rows.to(DEV),
                         torch.tensor(c.pre, dtype=torch.int64, device=DEV), plan, c.ps, c.Hq, max(c.len), **kw)


def want(c, parents, softcap=0.0, slopes=None, window=0):
    outs, tols = [], []
    for b, par in enumerate(parents):
        seen, depth = ancestors_ref(par)
        P, a = c.pre[b], c.cu[b]
        rows = []
        for j in range(len(par)):
            up = sorted(seen[j])
            keys = [(k, k) for k in range(P)] + [(P + x, P + depth[x]) for x in up]                    # token, position
            keys = [(k, pos) for k, pos in keys if not window or pos > P + depth[j] - window]
            rows.append(([k for k, _ in keys], [pos for _, pos in keys], P + depth[j]))
        o, t = attend_ref(c.q[a:a + len(par)], c.k, c.v, c.slots[b], rows, c.dtype, c.D ** -0.5, softcap, slopes)
        outs.append(o), tols.append(t)
    return torch.cat(outs), torch.cat(tols)


@pytest.mark.parametrize("ps", [1, 3, 16])
@pytest.mark.parametrize("pages", [True, False], ids=["new-pages", "complete-table"])
def test_tree_metadata(ps, pages):
    pre, ext = [0, 1, 15, 16, 40, 7], [1, 33, 64, 5, 100, 0]
    c = Case(1, BF, (2, 1, 64), ps, pre, ext)
    parents = trees(2, ext, bad=True)
    full = c.table.clone()
    kw, table = {}, c.table.clone().to(DEV)
    if pages:
        fresh, off = [], [0]
        for b in range(c.B):
            first, last = -(-pre[b] // ps), -(-c.len[b] // ps)
            fresh += full[c.rows[b], first:last].tolist()
            off.append(len(fresh))
            table[c.rows[b], first:last] = -7
        kw = dict(new_pages=torch.tensor(fresh, dtype=torch.int32, device=DEV), new_page_off=torch.tensor(off, dtype=torch.int32, device=DEV))
    plan = prepare(c, parents, table=table, **kw)
    assert torch.equal(table.cpu(), full)
    mask = plan.mask.cpu().numpy().astype(np.int64) & 0xFFFFFFFF
    t = 0
    for b, par in enumerate(parents):
        seen, depth = ancestors_ref(par)
        for j in range(len(par)):
            assert {32 * w + x for w in range(mask.shape[1]) for x in range(32) if mask[t, w] >> x & 1} == seen[j]
            assert int(plan.positions[t]) == pre[b] + depth[j]
            assert int(plan.out_cache_loc[t]) == c.slots[b][pre[b] + j]
            t += 1


def test_tree_metadata_past_the_table():
    """Nodes past the table's width get no slot, and no page is entered beyond it."""
    from mi355_attn import _lib, ops
    table = torch.full((2, 6), 5, dtype=torch.int32, device=DEV)
    plan = ops.tree_prepare(table[:, :3], torch.tensor([1], device=DEV), torch.tensor([10], device=DEV), torch.arange(-1, 5, dtype=torch.int32, device=DEV),
                            torch.tensor([0, 6], dtype=torch.int32, device=DEV), 4, 6, new_pages=torch.tensor([9], dtype=torch.int32, device=DEV),
                            new_page_off=torch.tensor([0, 1], dtype=torch.int32, device=DEV))
    assert plan.out_cache_loc.tolist() == [22, 23] + [_lib.NO_SLOT] * 4
    assert bool((table == 5).all())


def test_page_offsets_past_the_list_read_nothing():
    """Offsets that contradict the list of new pages: no read leaves it, other requests are as they were."""
    from mi355_attn import ops
    table = torch.full((3, 8), 5, dtype=torch.int32, device=DEV)
    ops.tree_prepare(table, torch.tensor([0, 1], device=DEV), torch.tensor([8, 8], device=DEV), torch.tensor([-1, 0, -1, 0], dtype=torch.int32, device=DEV),
                     torch.tensor([0, 2, 4], dtype=torch.int32, device=DEV), 4, 2, new_pages=torch.tensor([9, 10], dtype=torch.int32, device=DEV),
                     new_page_off=torch.tensor([0, 1, 2 ** 30], dtype=torch.int32, device=DEV))
    assert table[:, 2].tolist() == [9, 10, 5] and bool((table[:, 3:] == 5).all())


def test_long_chain_and_largest_tree():
    n = 1024
    c = Case(3, BF, (1, 1, 64), 16, [5], [n])
    plan = prepare(c, [list(range(-1, n - 1))])
    assert torch.equal(plan.positions.cpu(), 5 + torch.arange(n))
    got = attn(c, plan).view(n, 1, 64)
    pick = [0, 1, 26, 27, 59, 500, 1023]                                   # a chain is a causal extend
    rows = [(list(range(5 + j + 1)), list(range(5 + j + 1)), 5 + j) for j in pick]
    check(got[pick], *attend_ref(c.q[pick], c.k, c.v, c.slots[0], rows, BF, 64 ** -0.5))


@pytest.mark.parametrize("mod", [dict(), dict(softcap=30.0), dict(slopes=True), dict(slopes=True, softcap=8.0)], ids=lambda m: "-".join(m) or "plain")
@pytest.mark.parametrize("dtype,heads,ps,pre,ext", [
    (BF, (4, 2, 64), 16, [0, 33, 100, 16], [1, 9, 33, 64]),
    (HF, (3, 1, 128), 1, [1, 31, 32, 63], [40, 2, 7, 5]),
    (BF, (8, 1, 128), 16, [2000, 5], [64, 3]),
    (HF, (2, 2, 64), 5, [700], [100]),
    (BF, (32, 8, 128), 16, [640], [8]),
])
def test_tree_attention(dtype, heads, ps, pre, ext, mod):
    c = Case(4, dtype, heads, ps, pre, ext)
    parents = trees(5, ext)
    kw = dict(mod)
    if "slopes" in kw:
        kw["slopes"] = slopes_of(c.Hq)
    ref = want(c, parents, **kw)
    if "slopes" in kw:
        kw["slopes"] = kw["slopes"].to(DEV)
    got = attn(c, prepare(c, parents), **kw)
    check(got, *ref)
    assert torch.equal(got, attn(c, prepare(c, parents), **kw))


@pytest.mark.parametrize("window", [1, 3, 20, 64, 333, 2 ** 31 - 1])
@pytest.mark.parametrize("dtype,heads,ps,pre,ext,mod", [
    (BF, (4, 2, 64), 16, [0, 33, 100, 16], [1, 9, 33, 64], dict()),
    (HF, (3, 1, 128), 1, [1, 31, 900, 63], [5, 2, 4, 5], dict(slopes=True)),
    (BF, (8, 1, 128), 16, [2000, 5], [64, 3], dict(softcap=20.0)),
    (HF, (2, 2, 64), 5, [700], [8], dict()),
])
def test_tree_attention_in_a_window(dtype, heads, ps, pre, ext, mod, window):
    """A window counts positions, so nodes of one depth leave it together: windows shorter than a tree is deep drop ancestors."""
    c = Case(10, dtype, heads, ps, pre, ext)
    parents = trees(11, ext[:-1]) + [list(range(-1, ext[-1] - 1))]                                    # (the last one a chain)
    kw = dict(mod, window=window)
    if "slopes" in kw:
        kw["slopes"] = slopes_of(c.Hq)
    ref = want(c, parents, **kw)
    if "slopes" in kw:
        kw["slopes"] = kw["slopes"].to(DEV)
    check(attn(c, prepare(c, parents), **kw), *ref)


def test_siblings_do_not_leak():
    """NaN and infinities in one branch: its nodes say so, every other node is as if it were not there."""
    c = Case(6, BF, (4, 1, 64), 16, [50], [12])
    parents = [[-1, 0, 0, 1, 2, 3, 4, 2, 7, 0, 9, 10]]
    for x in (2, 7):                                                        # node 2's branch: 2, 4, 6, 7, 8
        c.v[c.slots[0][50 + x], 0, 3] = float("nan")
        c.v[c.slots[0][50 + x], 0, 9] = float("inf")
        c.k[c.slots[0][50 + x], 0, 1] = float("nan") if x == 7 else 1.0
    got = attn(c, prepare(c, parents)).view(12, 4, 64).double().cpu()
    ref, tol = want(c, parents)
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fine)
    assert bool(((got - ref).abs() <= tol)[fine].all())
    clean = [0, 1, 3, 5, 9, 10, 11]
    assert bool(fine[clean].all()) and not bool(fine[[2, 4, 6]].all())


def test_forest_without_a_prefix_and_masks_that_leave_nothing():
    from mi355_attn import ops
    c = Case(8, BF, (2, 1, 64), 4, [0, 0], [5, 3])
    parents = [[-1, -1, 0, 1, -1], [-1, 0, 1]]
    plan = prepare(c, parents)
    check(attn(c, plan), *want(c, parents))
    none = plan._replace(mask=torch.zeros_like(plan.mask))
    assert bool((attn(c, none) == 0).all())


def test_refusals():
    from mi355_attn import ops
    from mi355_attn._lib import MI355AttnError
    c = Case(9, BF, (2, 1, 64), 16, [5], [4])
    plan = prepare(c, [[-1, 0, 1, 2]])
    with pytest.raises(MI355AttnError, match="nodes"):
        attn(c, plan._replace(mask=plan.mask[:3]))
    with pytest.raises(MI355AttnError, match="positions"):
        attn(c, plan._replace(positions=plan.positions[:3]))
    with pytest.raises(MI355AttnError, match="1024"):
        ops.tree_prepare(c.table.to(DEV), c.rows.to(DEV), torch.tensor([5], device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV), plan.cu_q, 16, 2000)
    with pytest.raises(MI355AttnError, match="go together"):
        prepare(c, [[-1, 0, 1, 2]], new_pages=torch.zeros(1, dtype=torch.int32, device=DEV))
    with pytest.raises(MI355AttnError, match="parents"):
        ops.tree_prepare(c.table.to(DEV), c.rows.to(DEV), torch.tensor([5], device=DEV), torch.zeros(4, device=DEV), plan.cu_q, 16, 4)


def test_verification_step_replays_from_a_graph():
    """Metadata, attention and log probabilities of a step as one graph, replayed over other trees, prefixes and queries."""
    from mi355_attn import ops
    c = Case(41, BF, (8, 2, 64), 16, [600, 33, 90], [7, 7, 7])
    kp, vp, table, rows = c.pool(c.k), c.pool(c.v), c.table.to(DEV), c.rows.to(DEV)
    pre, cu = torch.tensor(c.pre, device=DEV), torch.tensor(c.cu, dtype=torch.int32, device=DEV)
    parents = torch.tensor([x for p in trees(1, [7, 7, 7]) for x in p], dtype=torch.int32, device=DEV)
    q = c.q.reshape(c.T, -1).to(DEV)
    head = torch.randn((512, 700), generator=c.g).to(DEV).to(BF)
    logits = torch.zeros((c.T, 700), dtype=BF, device=DEV)

    def step():
        plan = ops.tree_prepare(table, rows, pre, parents, cu, 16, 7)
        out = ops.tree_attn(q, kp, vp, table, rows, pre, plan, 16, 8, 700, softcap=20.0)
        torch.mm(out, head, out=logits)
        return plan.mask, plan.positions, plan.out_cache_loc, out, *ops.token_logprobs(logits, plan.positions % 700, top_k=3)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n in range(4):
        q.copy_(torch.randn(q.shape, generator=c.g).to(BF))
        pre.copy_(torch.tensor([600 - 97 * n, 33 - 8 * n, 90 - n]))
        parents.copy_(torch.tensor([x for p in trees(50 + n, [7, 7, 7]) for x in p], dtype=torch.int32))
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
