"""Layers with modified scores at the backend: which calls they make, and that a scale given to them is used."""
import itertools
from types import SimpleNamespace

import pytest
import torch

from oracle.scored_ref import attend_ref, visible_ref
from test_speculate import DEV, _engine, _rand, _slots

MODS = [dict(), dict(logit_cap=30.0), dict(window=8), dict(slopes=torch.ones(4)), dict(logit_cap=5.0, window=3)]


def test_layers_for_the_scored_kernels():
    """What decides in every layer of every step agrees with the options that are then passed on."""
    import mi355_attn as m
    from mi355_attn.backend import _any, _masks, _modified, _modifiers
    masks = [dict(), dict(doc_starts=torch.zeros(0, dtype=torch.int32)), dict(bidir_lens=torch.zeros(2, dtype=torch.int32))]
    for mod, mask in itertools.product(MODS, masks):
        layer, batch = m.Attention(0, 4, 2, 64, scale=0.3, **mod), SimpleNamespace(**mask)
        assert _modified(layer, batch) == bool(mod or mask) == (_any(_modifiers(layer)) or _any(_masks(batch)))
    assert not _modified(SimpleNamespace(layer_id=0, scale=0.5), SimpleNamespace())


@pytest.mark.parametrize("tree", [False, True], ids=["extend", "tree"])
def test_a_given_scale_is_passed_on(monkeypatch, tree):
    """Only by layers with modified scores: without any, the scale is the reference's, which no backend uses."""
    import mi355_attn as m
    from mi355_attn import backend
    seen = []
    monkeypatch.setattr(backend.ops, "scored_workspace_bytes", lambda *a: 0)
    monkeypatch.setattr(backend.ops, "scored_attn", lambda *a, **kw: seen.append(kw["scale"]))
    monkeypatch.setattr(backend.ops, "tree_attn", lambda *a, **kw: seen.append(kw["scale"]))
    be = backend.MI355AttnBackend(SimpleNamespace(device="cpu", page_size=4))
    lens = torch.tensor([3])
    batch = SimpleNamespace(mode=m.Mode.TREE if tree else m.Mode.PREFILL, tree=SimpleNamespace(max_nodes=3) if tree else None, tree_lens_host=[6],
                            seq_lens=lens, seq_lens_host=[3], prefix_lens=lens - 3, prefix_lens_host=[0], cu_q=torch.tensor([0, 3]),
                            kvcache=SimpleNamespace(get_kv_cache=lambda i: (None, None)), page_manager=SimpleNamespace(page_table=None), page_table_ids=None)
    q = torch.zeros(3, 256)
    for mod in MODS[1:]:
        for scale in (None, 1.0, 0.0625):
            be.forward(q, None, None, m.Attention(0, 4, 2, 64, scale, **mod), batch)
            assert seen.pop() == scale
    batch.doc_starts = None if tree else torch.zeros(3, dtype=torch.int32)
    be.forward(q, None, None, m.Attention(0, 4, 2, 64, 0.0625), batch)
    assert seen.pop() is None
    assert m.Attention(0, 4, 2, 64).scale == 1.0 and m.Attention(0, 4, 2, 64, 0.25).scale == 0.25


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1.0, 144 ** -0.5])
def test_scaled_capped_layers_through_the_backend(scale):
    """Prefill, then a draft tree, then a decode step of a capped layer whose scale is not head_dim^-0.5."""
    import mi355_attn as m
    Hq, Hkv, D, ps, n = 8, 2, 128, 16, 45
    kv, pm, be, batch = _engine((Hq, Hkv, D), ps, [n])
    layer, g = m.Attention(0, Hq, Hkv, D, scale, logit_cap=50.0), torch.Generator().manual_seed(4)
    batch.attn_backend = be

    def step(T, rows):
        be.init_forward_metadata(batch)
        qkv = _rand(g, T, Hq, Hkv, D)
        got = layer(*(t for t in qkv.to(DEV).split([Hq * D, Hkv * D, Hkv * D], dim=-1)), batch).double().cpu().view(T, Hq, D)
        slots = _slots(pm, batch, 0, 1 + max(k for keys, _, _ in rows for k in keys), ps)
        want, tol = attend_ref(qkv[:, : Hq * D].view(T, Hq, D), kv.k_cache[0].cpu(), kv.v_cache[0].cpu(), slots, rows, torch.bfloat16, scale, 50.0)
        assert bool(((got - want).abs() <= tol).all())

    batch.prepare_for_prefill()
    step(n, [(visible_ref(t, n),) * 2 + (t,) for t in range(n)])
    batch.prepare_for_tree([[1, 2, 3]], [[-1, 0, 0]])
    step(3, [([*range(n + 1)],) * 2 + (n,), ([*range(n + 2)],) * 2 + (n + 1,), ([*range(n + 1), n + 2], [*range(n + 2)], n + 1)])
    batch.commit_tree([[0, 2]])
    batch.output_ids = torch.zeros(1, dtype=torch.int64, device=DEV)
    batch.prepare_for_decode()
    step(1, [([*range(n + 3)],) * 2 + (n + 2,)])


def test_a_tree_that_cannot_be_prepared_takes_no_pages(monkeypatch):
    """The metadata launch refuses (here for want of a GPU): pages and mode are as they were, and the next step can begin."""
    import mi355_attn as m
    from test_speculate import _cpu_batch
    b, kv = _cpu_batch()
    b.mode, b.seq_lens, b.page_table_ids = m.Mode.DECODE, torch.tensor([6, 8]), torch.tensor([0, 1])
    before, table = sorted(kv.free_pages), b.page_manager.page_table.clone()
    for _ in range(8):                                                     # (more often than the pool has room for)
        with pytest.raises(RuntimeError, match="GPU"):
            b.prepare_for_tree([[1] * 9, [2] * 5], [list(range(-1, 8)), [-1] * 5])
        assert sorted(kv.free_pages) == before and b.tree is None and b.mode is m.Mode.DECODE
    assert torch.equal(b.page_manager.page_table, table)
