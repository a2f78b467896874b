"""Scored layers, draft trees and log probabilities together, as an engine runs them: Batch.prepare_for_tree / commit_tree, the
backend's dispatch, and speculative decoding on the harness runner.  Host logic on the CPU, everything else on the GPU."""
import math

import numpy as np
import pytest
import torch

from oracle.scored_ref import ancestors_ref, attend_ref, visible_ref

DEV = "cuda"


# ------------------------------------------------------------------------------------------------ host logic
def test_history_tree_and_path():
    from harness.speculate import accepted_path, history_tree
    tokens, parents = history_tree([1, 2, 3, 4, 1, 2, 5, 1], 8, depth=3)
    # occurrences of 1, the latest first: 2 5 1, then 2 3 4, sharing the 2
    assert tokens == [1, 2, 5, 1, 3, 4] and parents == [-1, 0, 1, 2, 1, 4]
    assert history_tree([9, 8, 7], 8) == ([7], [-1])
    assert len(history_tree([1, 2] * 50, 5)[0]) == 5
    tree = (tokens, parents)
    assert accepted_path(tree, [2, 3, 0, 0, 4, 0]) == [0, 1, 4, 5]
    assert accepted_path(tree, [9, 0, 0, 0, 0, 0]) == [0]


def _cpu_batch(pages=20, ps=4, lens=(6, 8)):
    import mi355_attn as m
    kv = m.KVCache(size=pages * ps, page_size=ps, head_num=1, head_dim=8, dtype=torch.bfloat16, layer_num=1, device="cpu")
    pm = m.PageManager(page_size=ps, max_req_num=4, max_context_len=64, device="cpu")
    b = m.Batch([m.Req(i, list(range(n))) for i, n in enumerate(lens)], pm, kv, device="cpu")
    b.seq_lens_host = list(lens)
    return b, kv


def test_prepare_for_tree_refuses_before_it_takes_anything():
    b, kv = _cpu_batch()
    before = kv.free_pages
    for ids, par in (([[1]], [[-1]]), ([[1], [2, 3]], [[-1], [-1]]), ([[1], []], [[-1], []]), ([[1], [2, 3]], [[-1], [-1, 1]]),
                     ([[1], [2, 3]], [[-1], [-2, 0]]), ([[0] * 1025, [1]], [[-1] * 1025, [-1]])):
        with pytest.raises(ValueError):
            b.prepare_for_tree(ids, par)
    with pytest.raises(RuntimeError, match="columns"):
        b.prepare_for_tree([[0] * 60, [1]], [[-1] * 60, [-1]])
    with pytest.raises(RuntimeError, match="exhausted"):
        _b, _kv = _cpu_batch(pages=3)
        _b.prepare_for_tree([[0] * 20, [1]], [[-1] * 20, [-1]])
    assert kv.free_pages == before and b.tree is None
    with pytest.raises(RuntimeError, match="no tree"):
        b.commit_tree([[0], [0]])


def test_dispatch_of_layers_and_masks():
    """Reference layers and plain layers stay on the paths they had; modifiers and masks are seen."""
    from types import SimpleNamespace

    import mi355_attn as m
    from mi355_attn.backend import _any, _masks, _modifiers
    assert not _any(_modifiers(SimpleNamespace(layer_id=0))) and not _any(_modifiers(m.Attention(0, 4, 2, 64)))
    assert _any(_modifiers(m.Attention(0, 4, 2, 64, logit_cap=30.0))) and _any(_modifiers(m.Attention(0, 4, 2, 64, window=8)))
    assert _any(_modifiers(m.Attention(0, 4, 2, 64, slopes=torch.zeros(4))))
    assert not _any(_masks(SimpleNamespace())) and _any(_masks(SimpleNamespace(doc_starts=torch.zeros(0, dtype=torch.int32), bidir_lens=None)))


def test_bench_modes_exclude_each_other():
    import bench_one_batch as bob
    for kw in (dict(graph=True, speculate=4), dict(graph=True, top_logprobs=2), dict(speculate=4, top_logprobs=2)):
        with pytest.raises(ValueError, match="one of"):
            bob.latency_test(None, bob.BenchArgs(**kw), 1, 8, 4, print, 1)


def test_a_request_that_is_done_keeps_nothing_more(monkeypatch):
    """Requests of a batch advance at their own pace: one that has its tokens must not fill the cache while the others go on."""
    from types import SimpleNamespace

    from harness import speculate
    nxt = lambda t: (7 * t + 3) % 50  # noqa: E731
    kept, held = [0, 0], []

    class FakeBatch:
        reqs = [SimpleNamespace(origin_input_ids=[1, 2]), SimpleNamespace(origin_input_ids=[5])]

        def prepare_for_tree(self, ids, parents):
            self.ids = ids
            held.append([k + len(i) for k, i in zip(kept, ids)])

        def commit_tree(self, paths):
            for b, path in enumerate(paths):
                kept[b] += len(path)

    def logprobs(logits, top_k):
        return SimpleNamespace(top_ids=logits.argmax(1, keepdim=True), top_logprobs=logits.max(1, keepdim=True).values)

    monkeypatch.setattr(speculate.m.ops, "token_logprobs", logprobs)
    forward = lambda batch: (torch.nn.functional.one_hot(torch.tensor([nxt(t) for i in batch.ids for t in i]), 50).float(), None)  # noqa: E731

    def draft(history, nodes):
        chain = [history[-1]]
        while history[0] == 1 and len(chain) < nodes:                      # the first request's drafts are all right
            chain.append(nxt(chain[-1]))
        return chain, list(range(-1, len(chain) - 1))

    out, lps, steps = speculate.speculative_decode(SimpleNamespace(forward=forward), torch.tensor([4, 6]), FakeBatch(), 10, 5, draft)
    for ids, first in zip(out, (4, 6)):
        want = [nxt(first)]
        while len(want) < 10:
            want.append(nxt(want[-1]))
        assert ids == want
    assert steps == 10 and kept == [10, 10] and max(max(h) for h in held) <= 11 and all(len(x) == 10 for x in lps)


# ------------------------------------------------------------------------------------------------ GPU
def _engine(heads, ps, lens, dtype=torch.bfloat16, layers=2, extra=200):
    import mi355_attn as m
    from types import SimpleNamespace
    Hq, Hkv, D = heads
    pages = sum(-(-(n + extra) // ps) for n in lens) + 4
    kv = m.KVCache(pages * ps, ps, Hkv, D, dtype, layers, DEV, device_free_list=True)
    kv.set_free_pages(torch.randperm(pages, generator=torch.Generator().manual_seed(3)).tolist())
    pm = m.PageManager(ps, len(lens) + 2, max(lens) + extra + ps, DEV)
    be = m.MI355AttnBackend(SimpleNamespace(device=DEV, page_size=ps, kvcache=kv, page_manager=pm))
    reqs = [m.Req(i, list(range(n))) for i, n in enumerate(lens)]
    for r in reqs:
        r.fill_ids = list(r.origin_input_ids)
    return kv, pm, be, m.Batch(reqs, pm, kv, device=DEV)


def _rand(g, T, Hq, Hkv, D):
    return (torch.randn((T, (Hq + 2 * Hkv) * D), generator=g) * 2).to(torch.bfloat16)


def _slots(pm, batch, b, n, ps):
    row = pm.page_table[int(batch.page_table_ids[b])].cpu()
    return [int(row[t // ps]) * ps + t % ps for t in range(n)]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,mods", [((6, 2, 64), dict(logit_cap=20.0, slopes=True)), ((8, 1, 128), dict(window=19)), ((4, 4, 64), dict()),
                                        ((5, 1, 64), dict(logit_cap=15.0))], ids=["cap-bias-g3", "window-g8", "masks-only", "cap-g5"])
def test_backend_prefill_then_decode_with_modified_scores(heads, mods):
    import mi355_attn as m
    Hq, Hkv, D = heads
    ps, lens = 16, [33, 5, 70]
    kv, pm, be, batch = _engine(heads, ps, lens)
    g = torch.Generator().manual_seed(1)
    slopes = torch.tensor([2.0 ** (-i - 1) for i in range(Hq)]) if "slopes" in mods else None
    layer = m.Attention(1, Hq, Hkv, D, logit_cap=mods.get("logit_cap", 0.0), window=mods.get("window", 0), slopes=None if slopes is None else slopes.to(DEV))
    batch.prepare_for_prefill()
    docs = [t // 20 * 20 for n in lens for t in range(n)] if not mods else None
    if docs:
        batch.doc_starts = torch.tensor(docs, dtype=torch.int32, device=DEV)
        batch.bidir_lens = torch.tensor([8, 0, 30], dtype=torch.int32, device=DEV)
    at = np.concatenate([[0], np.cumsum(lens)])

    def compare(got, q, rows):
        kp, vp = kv.k_cache[1].cpu(), kv.v_cache[1].cpu()
        for b, vis in enumerate(rows):
            a, e = (at[b], at[b + 1]) if len(rows[0]) > 1 else (b, b + 1)
            n = max(k for keys, _, _ in vis for k in keys) + 1
            want, tol = attend_ref(q[a:e].view(-1, Hq, D), kp, vp, _slots(pm, batch, b, n, ps), vis, torch.bfloat16, D ** -0.5,
                                   mods.get("logit_cap", 0.0), slopes)
            assert bool(((got[a:e].double().cpu().view(want.shape) - want).abs() <= tol).all())

    qkv = _rand(g, sum(lens), Hq, Hkv, D)
    q, k, v = qkv.to(DEV).split([Hq * D, Hkv * D, Hkv * D], dim=-1)
    be.init_forward_metadata(batch)
    batch.attn_backend = be
    got = layer(q, k, v, batch)
    rows = []
    for b, n in enumerate(lens):
        vis = []
        for t in range(n):
            keys = visible_ref(t, n, mods.get("window", 0), docs[at[b] + t] if docs else 0, [8, 0, 30][b] if docs else 0)
            vis.append((keys, keys, t))
        rows.append(vis)
    compare(got, qkv[:, : Hq * D], rows)
    for step in range(2):
        batch.output_ids = torch.zeros(3, dtype=torch.int64, device=DEV)
        batch.prepare_for_decode()
        assert batch.doc_starts is None and batch.bidir_lens is None
        qkv = _rand(g, 3, Hq, Hkv, D)
        q, k, v = qkv.to(DEV).split([Hq * D, Hkv * D, Hkv * D], dim=-1)
        be.init_forward_metadata(batch)
        got = layer(q, k, v, batch)
        rows = [[(visible_ref(n + step, n + step + 1, mods.get("window", 0)),) * 2 + (n + step,)] for n in lens]
        compare(got, qkv[:, : Hq * D], rows)


@pytest.mark.gpu
@pytest.mark.parametrize("ps", [1, 4, 16])
def test_tree_step_then_commit_then_decode(ps):
    """Prefill, verify a tree, keep a path, verify again, decode: pools, page table, free pages and outputs at every step."""
    import mi355_attn as m
    Hq, Hkv, D = 4, 2, 64
    lens = [15, 4, 33]
    kv, pm, be, batch = _engine((Hq, Hkv, D), ps, lens)
    layer = m.Attention(0, Hq, Hkv, D)
    g = torch.Generator().manual_seed(2)
    batch.prepare_for_prefill()
    qkv = _rand(g, sum(lens), Hq, Hkv, D)
    be.init_forward_metadata(batch)
    batch.attn_backend = be
    be.forward(*(t for t in qkv.to(DEV).split([Hq * D, Hkv * D, Hkv * D], dim=-1)), layer, batch)
    at = np.concatenate([[0], np.cumsum(lens)])
    keys = [[qkv[t, Hq * D:(Hq + Hkv) * D].view(Hkv, D) for t in range(at[b], at[b + 1])] for b in range(3)]      # what the cache holds
    vals = [[qkv[t, (Hq + Hkv) * D:].view(Hkv, D) for t in range(at[b], at[b + 1])] for b in range(3)]
    trees = [([-1, 0, 0, 1, 3, 2], [[0, 1, 3, 4]]), ([-1, 0, 1, 1, 0], [[0, 4]]), ([-1] + [0] * 18 + [18], [[0, 18, 19]])]
    for _round in range(2):
        held = list(batch.seq_lens_host)
        free = kv.available_page_num()
        parents = [p for p, _ in trees]
        T = sum(len(p) for p in parents)
        batch.prepare_for_tree([[7] * len(p) for p in parents], parents)
        with pytest.raises(RuntimeError, match="open"):
            batch.prepare_for_decode()
        be.init_forward_metadata(batch)
        qkv = _rand(g, T, Hq, Hkv, D)
        q, k, v = qkv.to(DEV).split([Hq * D, Hkv * D, Hkv * D], dim=-1)
        got = be.forward(q, k, v, layer, batch).double().cpu().view(T, Hq, D)
        assert torch.equal(kv.k_cache[0][batch.out_cache_loc].cpu().reshape(T, -1), qkv[:, Hq * D:(Hq + Hkv) * D])
        first = 0
        for b, par in enumerate(parents):
            seen, depth = ancestors_ref(par)
            P, n = held[b], len(par)
            kk = torch.stack(keys[b] + [qkv[first + j, Hq * D:(Hq + Hkv) * D].view(Hkv, D) for j in range(n)])
            vv = torch.stack(vals[b] + [qkv[first + j, (Hq + Hkv) * D:].view(Hkv, D) for j in range(n)])
            vis = []
            for j in range(n):
                ks = list(range(P)) + [P + x for x in sorted(seen[j])]
                vis.append((ks, ks, P + depth[j]))
            want, tol = attend_ref(qkv[first:first + n, : Hq * D].view(n, Hq, D), kk, vv, range(P + n), vis, torch.bfloat16, D ** -0.5)
            assert bool(((got[first:first + n] - want).abs() <= tol).all())
            assert batch.positions[first:first + n].tolist() == [P + d for d in depth]
            path = trees[b][1][0]
            keys[b] += [kk[P + j] for j in path]
            vals[b] += [vv[P + j] for j in path]
            first += n
        with pytest.raises(ValueError):
            batch.commit_tree([[0, 4], [0], [0]])
        batch.commit_tree([t[1][0] for t in trees])
        assert batch.seq_lens_host == [p + len(t[1][0]) for p, t in zip(held, trees)] == batch.seq_lens.tolist()
        used = sum(-(-n // ps) - -(-p // ps) for n, p in zip(batch.seq_lens_host, held))
        assert kv.available_page_num() == free - used and kv.ring.snapshot() == kv.free_pages
        for b in range(3):
            slots = _slots(pm, batch, b, batch.seq_lens_host[b], ps)
            assert len(set(slots)) == len(slots) and not {s // ps for s in slots} & set(kv.free_pages)
            assert torch.equal(kv.k_cache[0][slots].cpu(), torch.stack(keys[b])) and torch.equal(kv.v_cache[0][slots].cpu(), torch.stack(vals[b]))
    batch.output_ids = torch.zeros(3, dtype=torch.int64, device=DEV)
    batch.prepare_for_decode()
    be.init_forward_metadata(batch)
    qkv = _rand(g, 3, Hq, Hkv, D)
    got = be.forward(*(t for t in qkv.to(DEV).split([Hq * D, Hkv * D, Hkv * D], dim=-1)), layer, batch).double().cpu().view(3, Hq, D)
    for b in range(3):
        kk = torch.stack(keys[b] + [qkv[b, Hq * D:(Hq + Hkv) * D].view(Hkv, D)])
        vv = torch.stack(vals[b] + [qkv[b, (Hq + Hkv) * D:].view(Hkv, D)])
        n = kk.shape[0]
        want, tol = attend_ref(qkv[b:b + 1, : Hq * D].view(1, Hq, D), kk, vv, range(n), [(list(range(n)),) * 2 + (n - 1,)], torch.bfloat16, D ** -0.5)
        assert bool(((got[b:b + 1] - want).abs() <= 2 * tol).all())     # (the plain decode kernel rounds as the scored one does)


@pytest.mark.gpu
def test_trees_in_windowed_layers():
    import mi355_attn as m
    Hq, Hkv, D, ps, W = 4, 2, 64, 16, 12
    kv, pm, be, batch = _engine((Hq, Hkv, D), ps, [40])
    layer, g = m.Attention(0, Hq, Hkv, D, window=W, logit_cap=15.0), torch.Generator().manual_seed(8)
    batch.prepare_for_prefill()
    be.init_forward_metadata(batch)
    qkv = _rand(g, 40, Hq, Hkv, D)
    be.forward(*(t for t in qkv.to(DEV).split([Hq * D, Hkv * D, Hkv * D], dim=-1)), layer, batch)
    parents = [[*range(-1, 14), 3, 15, 0]]                                  # a chain longer than the window, two branches
    batch.prepare_for_tree([[7] * 18], parents)
    be.init_forward_metadata(batch)
    new = _rand(g, 18, Hq, Hkv, D)
    got = be.forward(*(t for t in new.to(DEV).split([Hq * D, Hkv * D, Hkv * D], dim=-1)), layer, batch).double().cpu().view(18, Hq, D)
    both = torch.cat([qkv, new])
    seen, depth = ancestors_ref(parents[0])
    rows = []
    for j in range(18):
        keys = [(k, k) for k in range(40)] + [(40 + x, 40 + depth[x]) for x in sorted(seen[j])]
        keys = [(k, pos) for k, pos in keys if pos > 40 + depth[j] - W]
        rows.append(([k for k, _ in keys], [pos for _, pos in keys], 40 + depth[j]))
    want, tol = attend_ref(new[:, : Hq * D].view(18, Hq, D), both[:, Hq * D:(Hq + Hkv) * D].view(58, Hkv, D), both[:, (Hq + Hkv) * D:].view(58, Hkv, D),
                           range(58), rows, torch.bfloat16, D ** -0.5, 15.0)
    assert bool(((got - want).abs() <= tol).all())


@pytest.mark.gpu
def test_trees_take_no_masks():
    import mi355_attn as m
    kv, pm, be, batch = _engine((4, 2, 64), 16, [5])
    batch.prepare_for_prefill()
    batch.prepare_for_tree([[1, 2]], [[-1, 0]])
    batch.doc_starts = torch.zeros(2, dtype=torch.int32, device=DEV)
    be.init_forward_metadata(batch)
    z = torch.zeros((2, 4 * 64), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="mask"):
        be.forward(z, z[:, :128], z[:, :128], m.Attention(0, 4, 2, 64), batch)
    batch.commit_tree([[0]])
    assert batch.doc_starts is None and batch.seq_lens_host == [6]


@pytest.mark.gpu
@pytest.mark.parametrize("model,ps", [("tiny", 16), ("tiny-capped", 4), ("tiny128", 1), ("tiny-window", 16)])
def test_speculative_decode_runs_and_agrees(model, ps):
    """Drafts that are right (the plain loop's own tokens, among wrong ones): few steps, the plain loop's tokens, and log
    probabilities that are those of its logits."""
    import bench_one_batch as bob
    from harness.llama_shell import SHAPES, HarnessRunner
    from harness.speculate import speculative_decode
    from mi355_attn import ops
    shape, B, L, n = SHAPES[model], 3, 40, 12
    runner = HarnessRunner(shape, ps, max_total_tokens=B * (L + 80) + 64 * ps, max_reqs=B, context_len=L + 80)
    prompts = [p[: L - 3 * i] for i, p in enumerate(bob.synth_prompts(B, L, shape.vocab, seed=5))]
    first, logits0, batch = bob.extend(bob.make_reqs(prompts), runner)
    nxt, plain, plain_lp, margin = first, [], [], []
    for _ in range(n):
        nxt, logits = bob.decode(nxt, batch, runner)
        two = torch.topk(logits.float(), 2).values
        margin.append((two[:, 0] - two[:, 1]).cpu())
        plain.append(nxt.cpu())
        plain_lp.append(ops.token_logprobs(logits, nxt).logprobs.cpu())
    plain, plain_lp, margin = torch.stack(plain, 1), torch.stack(plain_lp, 1), torch.stack(margin, 1)
    bob.reset_pools(runner)
    first2, _, batch = bob.extend(bob.make_reqs(prompts), runner)
    assert torch.equal(first, first2)
    known = [prompts[b] + [int(first[b])] + plain[b].tolist() for b in range(B)]

    def draft(history, nodes):
        b = next(i for i in range(B) if history[: len(prompts[i])] == prompts[i] and len(history) > len(prompts[i]))
        right = known[b][len(history): len(history) + 3] if history == known[b][: len(history)] else []
        tokens, parents = [history[-1]], [-1]
        for tok in right:
            if len(tokens) + 2 > max(nodes, 2):
                break
            tokens += [(tok + 1) % shape.vocab, tok]
            parents += [0 if len(parents) == 1 else len(parents) - 1] * 2
        return tokens, parents

    toks, lps, steps = speculative_decode(runner, first2, batch, n, 7, draft=draft)
    toks, lps = torch.tensor(toks), torch.tensor(lps)
    scale = float(logits0.float().abs().max())
    for b in range(B):
        # (equal as long as the plain loop's choice was clearer than the two forms' difference in rounding)
        clear = (margin[b] > 0.05 * scale).int().cumprod(0).bool()
        assert torch.equal(toks[b][clear], plain[b][clear])
        same = (toks[b] == plain[b]).int().cumprod(0).bool()
        assert bool(((lps[b] - plain_lp[b]).abs()[same] <= 0.1 * scale).all())
    if bool((toks == plain).all()):
        assert steps <= math.ceil(n / 2)


@pytest.mark.gpu
@pytest.mark.parametrize("model", ["tiny-capped", "tiny-window"])
def test_three_phase_with_modified_scores(model):
    """prefill(cut) -> extend over the cached prefix -> decode against a single shot, through capped, biased, windowed layers;
    the decode loop replayed from a captured graph gives the eager loop's tokens."""
    import bench_one_batch as bob
    from harness.llama_shell import SHAPES, HarnessRunner
    shape, ps, B, L, out_len, cut = SHAPES[model], 16, 3, 90, 8, 48
    runner = HarnessRunner(shape, ps, max_total_tokens=B * 2 * (L + out_len + 2 * ps) + 64 * ps, max_reqs=B, context_len=L + out_len + ps)
    prompts = [p[:n] for p, n in zip(bob.synth_prompts(B, L, shape.vocab, seed=3), (90, 61, 77))]
    logits3, ids3 = bob.three_phase(runner, prompts, cut, out_len)
    bob.reset_pools(runner)
    logits1, ids1 = bob.three_phase(runner, prompts, 0, out_len)
    scale = float(logits1.float().abs().max())
    assert torch.isfinite(logits3).all() and scale > 0
    assert float((logits3.float() - logits1.float()).abs().max()) <= 0.05 * scale
    bob.reset_pools(runner)
    _, graphed = bob.three_phase(runner, prompts, 0, out_len, graph=True)
    assert torch.equal(graphed, ids1)


@pytest.mark.gpu
def test_bench_modes_run():
    import bench_one_batch as bob
    from harness.llama_shell import SHAPES, HarnessRunner
    runner = HarnessRunner(SHAPES["tiny"], 16, max_total_tokens=8192, max_reqs=2, context_len=256)
    quiet = lambda *a, **k: None  # noqa: E731
    res = bob.latency_test(runner, bob.BenchArgs(model="tiny", top_logprobs=5), 2, 64, 6, quiet, 1)
    assert res["top_logprobs"] == 5 and res["decode_throughput"] > 0
    res = bob.latency_test(runner, bob.BenchArgs(model="tiny", speculate=6), 2, 64, 9, quiet, 1)
    assert 1 <= res["speculative_steps"] <= 8 and res["decode_throughput"] > 0
    said = []
    bob.correctness_test(runner, bob.BenchArgs(model="tiny", batch_size=(2,), input_len=(60,), output_len=(6,), cut_len=16, speculate=6), said.append)
    assert any("speculative decode" in s for s in said)
