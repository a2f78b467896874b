"""m355_scored_attn on the GPU against the definition in 64 bits (oracle/scored_ref.py, which derives the bounds)."""
import numpy as np
import pytest
import torch

from oracle.scored_ref import attend_ref, visible_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


class Case:
    """A batch on the host: lengths, shuffled pages, pools with NaN in every slot that no request uses."""

    def __init__(self, seed, dtype, heads, ps, pre, ext, pad=0, width_extra=2, amp=2.0, shared=False):
        self.g = torch.Generator().manual_seed(seed)
        self.dtype, (self.Hq, self.Hkv, self.D), self.ps = dtype, heads, ps
        self.pre, self.ext = list(pre), list(ext)
        self.len = [p + e for p, e in zip(pre, ext)]
        self.B, self.T = len(pre), sum(ext)
        self.cu = np.concatenate([[0], np.cumsum(ext)]).tolist()
        pages = [-(-n // ps) for n in self.len]
        total = sum(pages) + 3
        perm = torch.randperm(total, generator=self.g)
        W = max(pages + [1]) + width_extra
        self.table = torch.full((self.B + 2, W), 2 ** 31 - 1, dtype=torch.int32)            # entries past a request: garbage
        self.rows = torch.randperm(self.B + 2, generator=self.g)[: self.B]
        at = 0
        for b in range(self.B):
            self.table[self.rows[b], : pages[b]] = perm[at:at + pages[b]].int()
            at += pages[b]
        self.slots = [[int(self.table[self.rows[b], t // ps]) * ps + t % ps for t in range(self.len[b])] for b in range(self.B)]
        S = total * ps
        used = torch.zeros(S, dtype=torch.bool)
        for s in self.slots:
            used[s] = True
        self.k = torch.randn((S, self.Hkv, self.D), generator=self.g).to(dtype)
        self.v = torch.randn((S, self.Hkv, self.D), generator=self.g).to(dtype)
        self.k[~used], self.v[~used] = float("nan"), float("nan")
        self.q = (torch.randn((self.T, self.Hq, self.D), generator=self.g) * amp).to(dtype)
        self.pad = pad

    def pool(self, x):
        S = x.shape[0]
        full = torch.full((S, self.Hkv * self.D + self.pad), float("nan"), dtype=self.dtype, device=DEV)
        full[:, : self.Hkv * self.D] = x.reshape(S, -1).to(DEV)
        return full[:, : self.Hkv * self.D].unflatten(1, (self.Hkv, self.D))

    def run(self, decode=False, q=None, table=None, **kw):
        from mi355_attn import ops
        if not decode:
            kw = dict(prefix_lens=torch.tensor(self.pre, device=DEV), cu_q=torch.tensor(self.cu, dtype=torch.int32, device=DEV),
                      max_extend_len=max(self.ext), **kw)
        q = self.q.reshape(self.T, -1).to(DEV) if q is None else q
        return ops.scored_attn(q, self.pool(self.k), self.pool(self.v), self.table.to(DEV) if table is None else table, self.rows.to(DEV),
                               torch.tensor(self.len, dtype=torch.int64, device=DEV), self.ps, self.Hq, max(max(self.len), 1), **kw)

    def want(self, softcap=0.0, slopes=None, window=0, doc_starts=None, bidir=None, rows=None):
        outs, tols = [], []
        for b in range(self.B):
            a = self.cu[b]
            js = range(self.ext[b]) if rows is None else [j for j in rows if j < self.ext[b]]
            vis = []
            for j in js:
                pos = self.pre[b] + j
                keys = visible_ref(pos, self.len[b], window, 0 if doc_starts is None else int(doc_starts[a + j]), 0 if bidir is None else int(bidir[b]))
                vis.append((keys, keys, pos))
            o, t = attend_ref(self.q[[a + j for j in js]], self.k, self.v, self.slots[b], vis, self.dtype, self.D ** -0.5, softcap, slopes)
            outs.append(o), tols.append(t)
        return torch.cat(outs), torch.cat(tols)


def check(got, want, tol):
    got = got.double().cpu().view(want.shape)
    assert torch.isfinite(got).all(), "masked places reached the output"
    off = (got - want).abs() - tol
    assert float(off.max()) <= 0, f"{float(off.max())} over the bound at {np.unravel_index(int(off.argmax()), off.shape)}"


def slopes_of(Hq):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / Hq) for i in range(Hq)], dtype=torch.float32)


SHAPES = [  # dtype, heads, page size, prefix lengths, new tokens, row padding
    (BF, (4, 2, 64), 16, [0, 33, 0, 17, 5], [1, 70, 40, 2, 33], 0),
    (HF, (3, 1, 128), 1, [0, 1, 31, 32], [3, 1, 33, 64], 8),
    (BF, (5, 5, 128), 3, [10, 100], [9, 35], 64),
    (HF, (8, 1, 64), 64, [300, 0, 64], [20, 129, 1], 0),
    (BF, (16, 1, 128), 16, [40, 7], [11, 30], 0),
]
MODS = [dict(), dict(softcap=30.0), dict(slopes=True), dict(softcap=5.0, slopes=True, window=20), dict(window=1), dict(window=37),
        dict(doc=True), dict(bidir=True), dict(doc=True, bidir=True, slopes=True, softcap=50.0)]


@pytest.mark.parametrize("mod", MODS, ids=lambda m: "-".join(m) or "plain")
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_extend(shape, mod):
    dtype, heads, ps, pre, ext, pad = SHAPES[shape]
    c = Case(shape, dtype, heads, ps, pre, ext, pad)
    kw, ref = dict(softcap=mod.get("softcap", 0.0), window=mod.get("window", 0)), dict(softcap=mod.get("softcap", 0.0), window=mod.get("window", 0))
    if "slopes" in mod:
        ref["slopes"] = slopes_of(c.Hq)
        kw["slopes"] = ref["slopes"].to(DEV)
    if "doc" in mod:
        # documents of 13 tokens; some rows name a start behind themselves: they see nothing (or the bidirectional part only)
        d = [(p + j) // 13 * 13 + (100000 if j % 7 == 3 else 0) for p, e in zip(pre, ext) for j in range(e)]
        ref["doc_starts"], kw["doc_starts"] = d, torch.tensor(d, dtype=torch.int32, device=DEV)
    if "bidir" in mod:
        b = [p + e // 2 for p, e in zip(pre, ext)]
        b[0] = 10 ** 6                                                   # longer than the request: all of it
        ref["bidir"], kw["bidir_lens"] = b, torch.tensor(b, dtype=torch.int32, device=DEV)
    check(c.run(**kw), *c.want(**ref))


@pytest.mark.parametrize("mod", [dict(), dict(softcap=50.0), dict(slopes=True, softcap=20.0), dict(window=40), dict(doc=True)], ids=lambda m: "-".join(m) or "plain")
@pytest.mark.parametrize("dtype,heads,ps,pad", [(BF, (8, 2, 64), 16, 0), (HF, (8, 1, 128), 1, 64), (BF, (3, 3, 128), 5, 0), (HF, (12, 2, 64), 16, 0), (BF, (20, 1, 64), 16, 0)])
def test_single_token(dtype, heads, ps, pad, mod):
    lens = [1, 2, 31, 32, 33, 64, 65, 127, 500, 1025, 17]
    c = Case(7, dtype, heads, ps, [n - 1 for n in lens], [1] * len(lens), pad)
    kw, ref = dict(softcap=mod.get("softcap", 0.0), window=mod.get("window", 0)), dict(softcap=mod.get("softcap", 0.0), window=mod.get("window", 0))
    if "slopes" in mod:
        ref["slopes"] = slopes_of(c.Hq)
        kw["slopes"] = ref["slopes"].to(DEV)
    if "doc" in mod:
        ref["doc_starts"] = [n // 2 if i % 3 else n + 5 for i, n in enumerate(lens)]
        kw["doc_starts"] = torch.tensor(ref["doc_starts"], dtype=torch.int32, device=DEV)
    got = c.run(decode=True, **kw)
    check(got, *c.want(**ref))
    assert torch.equal(got, c.run(decode=True, **kw))                     # nothing depends on an order of arrival


@pytest.mark.parametrize("heads,B,L,mod", [((8, 1, 128), 1, 40001, dict(softcap=30.0)), ((4, 2, 64), 3, 9000, dict(slopes=True)),
                                           ((8, 8, 128), 2, 5000, dict(window=4097)), ((4, 1, 64), 40, 700, dict())])
def test_single_token_long(heads, B, L, mod):
    lens = [max(1, L - 977 * i) for i in range(B)]
    c = Case(11, BF, heads, 16, [n - 1 for n in lens], [1] * B)
    kw = dict(mod)
    if "slopes" in kw:
        kw["slopes"] = slopes_of(c.Hq)
    want = c.want(**kw)
    if "slopes" in kw:
        kw["slopes"] = kw["slopes"].to(DEV)
    check(c.run(decode=True, **kw), *want)


def test_short_turns_over_long_histories():
    c = Case(12, BF, (8, 2, 128), 16, [6000, 3001, 0, 900], [3, 20, 5, 40])
    check(c.run(softcap=40.0), *c.want(softcap=40.0))
    check(c.run(window=1000), *c.want(window=1000))


def test_long_extend_rows_sampled():
    c = Case(13, BF, (8, 2, 64), 16, [0, 77], [1400, 900])
    pick = [0, 1, 31, 32, 63, 127, 128, 500, 899, 1399]
    got = c.run(softcap=30.0).view(c.T, c.Hq, c.D)
    at = [c.cu[b] + j for b in range(2) for j in pick if j < c.ext[b]]
    check(got[at], *c.want(softcap=30.0, rows=pick))


def test_empty_requests_and_rows_behind_the_last():
    """Requests without rows, a request of length 0 in the single-token form, rows of a padded batch."""
    from mi355_attn import ops
    c = Case(14, BF, (4, 2, 64), 16, [5, 0, 40, 9], [3, 0, 0, 2])
    q = torch.cat([c.q.reshape(c.T, -1), torch.full((4, 256), float("nan"), dtype=BF)]).to(DEV)
    out = torch.full((c.T + 4, 256), 7.0, dtype=BF, device=DEV)
    c.run(q=q, out=out)
    check(out[: c.T], *c.want())
    assert bool((out[c.T:] == 7.0).all())
    lens = torch.tensor([0, 3], device=DEV)
    z = ops.scored_attn(c.q[:2].reshape(2, -1).to(DEV), c.pool(c.k), c.pool(c.v), c.table.to(DEV), c.rows[1:3].to(DEV), lens, 16, 4, 8)
    assert bool((z[0] == 0).all()) and bool(torch.isfinite(z[1]).all())
    empty = ops.scored_attn(c.q[:0].reshape(0, 256).to(DEV), c.pool(c.k), c.pool(c.v), c.table.to(DEV), c.rows[:0].to(DEV), lens[:0], 16, 4, 8)
    assert empty.shape == (0, 256)


@pytest.mark.parametrize("where", ["v", "k"])
@pytest.mark.parametrize("ext", [70, 1], ids=["extend", "single"])
def test_masked_nan_and_infinities_stay_out(where, ext):
    """Keys that some rows of a tile see and others do not hold NaN and infinities: rows that see them say so, the others must
    be as if nothing was there."""
    c = Case(15, BF, (4, 1, 128), 16, [80, 3], [ext, ext])
    bad = {0: [40, 79, 80 + ext // 2], 1: [0]}
    for b, toks in bad.items():
        for i, t in enumerate(toks):
            x = c.v if where == "v" else c.k
            x[c.slots[b][t], 0, 5 * i:5 * i + 3] = [float("nan"), float("inf"), -float("inf")][i]
    starts = [(0 if j % 3 == 0 else 41 + j % 5) if b == 0 else (2 if j % 2 or ext == 1 else 0) for b in range(2) for j in range(ext)]
    got = c.run(doc_starts=torch.tensor(starts, dtype=torch.int32, device=DEV)).view(c.T, c.Hq, c.D).double().cpu()
    want, tol = c.want(doc_starts=starts)
    same = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), same)
    assert bool(((got - want).abs() <= tol)[same].all())
    assert bool((~same).any()) and bool(same.any())


def test_scores_of_any_size():
    """Scores beyond every usual range: huge, all equal, -inf on every visible key of a row (zeros)."""
    c = Case(16, BF, (2, 1, 64), 16, [0], [40], amp=3000.0)
    got, (want, tol) = c.run(), c.want()
    # (weights are 0 or 1 almost everywhere here: a score's rounding decides nothing, the largest differ by far more than it)
    assert torch.isfinite(got).all()
    c.q.zero_()
    check(c.run(slopes=slopes_of(2).to(DEV)), *c.want(slopes=slopes_of(2)))
    c.q.fill_(1.0)
    c.k.fill_(-float("inf"))
    assert bool((c.run() == 0).all())


def test_strides_streams_and_views():
    """q out of a packed projection, out inside a wider buffer, a page table wider than it says, work on a side stream."""
    c = Case(17, HF, (6, 2, 64), 16, [33, 0], [17, 50], pad=64)
    W = c.Hq * c.D
    want = c.want(softcap=9.0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        packed = torch.full((c.T, W + 256), float("nan"), dtype=HF, device=DEV)
        packed[:, :W] = c.q.reshape(c.T, W).to(DEV)
        wide = torch.full((c.T, W + 64), 3.0, dtype=HF, device=DEV)
        table = torch.zeros((c.table.shape[0], c.table.shape[1] + 5), dtype=torch.int32, device=DEV)
        table[:, : c.table.shape[1]] = c.table.to(DEV)
        got = c.run(q=packed[:, :W], out=wide[:, :W], table=table[:, : c.table.shape[1]], softcap=9.0)
    side.synchronize()
    check(got, *want)
    assert bool((wide[:, W:] == 3.0).all())


def test_pool_past_32_bits():
    """A pool of more than 2^32 bytes whose used pages sit at its far end."""
    from mi355_attn import ops
    Hkv, D, ps, L = 8, 128, 16, 100
    S = (1 << 21) + 4096                                                  # 2 KiB rows
    k = torch.zeros((S, Hkv, D), dtype=BF, device=DEV)
    v = torch.zeros((S, Hkv, D), dtype=BF, device=DEV)
    g = torch.Generator().manual_seed(3)
    pages = [S // ps - 1 - i for i in range(-(-L // ps))]
    slots = [pages[t // ps] * ps + t % ps for t in range(L)]
    kh, vh = torch.randn((L, Hkv, D), generator=g).to(BF), torch.randn((L, Hkv, D), generator=g).to(BF)
    k[slots], v[slots] = kh.to(DEV), vh.to(DEV)
    q = torch.randn((1, 16, D), generator=g).to(BF)
    got = ops.scored_attn(q.view(1, -1).to(DEV), k, v, torch.tensor([pages], dtype=torch.int32, device=DEV),
                          torch.zeros(1, dtype=torch.int64, device=DEV), torch.tensor([L], device=DEV), ps, 16, L)
    keys = list(range(L))
    check(got, *attend_ref(q, kh, vh, keys, [(keys, keys, L - 1)], BF, D ** -0.5))


def test_bad_tables_read_nothing_outside():
    """Page ids far outside the pool inside a request's length: the result means nothing, but no read leaves the pools."""
    c = Case(18, BF, (4, 2, 64), 16, [30], [20])
    c.table[c.rows[0], 1] = 2 ** 31 - 1
    c.table[c.rows[0], 2] = -5
    c.k.nan_to_num_(), c.v.nan_to_num_()
    assert torch.isfinite(c.run()).all()


def test_captured_graph_replays():
    from mi355_attn import ops
    lens = [700, 33, 2100]
    c = Case(19, BF, (8, 2, 64), 16, [n - 1 for n in lens], [1] * 3)
    kp, vp, table, rows = c.pool(c.k), c.pool(c.v), c.table.to(DEV), c.rows.to(DEV)
    n = torch.tensor(lens, device=DEV)
    q = c.q.reshape(3, -1).to(DEV)
    ws = torch.empty(max(256, ops.scored_workspace_bytes(3, 3, 8, 2, 64, 1, 2100)), dtype=torch.uint8, device=DEV)
    call = lambda: ops.scored_attn(q, kp, vp, table, rows, n, 16, 8, 2100, softcap=30.0, workspace=ws)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step in range(4):
        q.copy_(torch.randn(q.shape, generator=c.g).to(BF))
        n.copy_(torch.tensor([700 - 30 * step, 33, 2100 - 500 * step]))
        eager = call().clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


@pytest.mark.parametrize("B,Hkv", [(130, 1), (70, 2), (300, 1)])
def test_more_requests_than_lanes(B, Hkv):
    """Batches of more requests than a wave has lanes, lengths from 1 to a few hundred, some requests without rows."""
    lens = [1 + (i * 37) % 311 for i in range(B)]
    c = Case(21, BF, (4 * Hkv, Hkv, 64), 16, [n - 1 for n in lens], [1] * B)
    check(c.run(decode=True, softcap=30.0), *c.want(softcap=30.0))
    ext = [0 if i % 9 == 0 else 1 + i % 6 for i in range(B)]
    c = Case(22, BF, (4 * Hkv, Hkv, 64), 16, [n - 1 for n in lens], ext)
    check(c.run(window=100), *c.want(window=100))


def test_hints_that_promise_too_little():
    """More rows per request than max_extend_len said: rows past it may be left out, nothing else suffers."""
    from mi355_attn import ops
    c = Case(23, BF, (4, 1, 64), 16, [40, 3], [30, 2])
    args = (c.q.reshape(c.T, -1).to(DEV), c.pool(c.k), c.pool(c.v), c.table.to(DEV), c.rows.to(DEV), torch.tensor(c.len, device=DEV), 16, 4)
    form = dict(prefix_lens=torch.tensor(c.pre, device=DEV), cu_q=torch.tensor(c.cu, dtype=torch.int32, device=DEV))
    want, tol = c.want()
    for ext, mx in ((2, 1), (4, 200), (30, 1)):
        got = ops.scored_attn(*args, mx, max_extend_len=ext, **form).double().cpu().view(want.shape)
        rows = [*range(min(ext, 30)), 30, 31]
        assert bool(((got - want).abs() <= tol)[rows].all()), (ext, mx)


def test_lengths_that_contradict_the_rows():
    """cu_q that runs backwards or past q, lengths past the table: in-bounds work, finite pools give finite rows or none."""
    from mi355_attn import ops
    c = Case(24, BF, (4, 2, 64), 16, [30, 5], [4, 4])
    c.k.nan_to_num_(), c.v.nan_to_num_()
    table = c.table.clamp(max=3)
    for cu, pre, lens in (([0, 4, 100], [30, 5], [34, 9]), ([4, 0, 8], [30, 5], [34, 9]), ([0, 4, 8], [-7, 2 ** 40], [2 ** 40, -3]), ([0, 0, 0], [1, 1], [1, 1])):
        out = torch.zeros((8, 256), dtype=BF, device=DEV)
        ops.scored_attn(c.q.reshape(8, -1).to(DEV), c.pool(c.k).nan_to_num(), c.pool(c.v).nan_to_num(), table.to(DEV), c.rows.to(DEV),
                        torch.tensor(lens, device=DEV), 16, 4, 40, prefix_lens=torch.tensor(pre, device=DEV),
                        cu_q=torch.tensor(cu, dtype=torch.int32, device=DEV), max_extend_len=8, out=out)
        torch.cuda.synchronize()


def test_refusals():
    from mi355_attn import MI355AttnBackend  # noqa: F401  (the package imports)
    from mi355_attn._lib import MI355AttnError
    c = Case(20, BF, (4, 2, 64), 16, [5, 6], [2, 3])
    i32 = dict(dtype=torch.int32, device=DEV)
    with pytest.raises(MI355AttnError, match="slopes"):
        c.run(slopes=torch.zeros(3, device=DEV))
    with pytest.raises(MI355AttnError, match="doc_starts"):
        c.run(doc_starts=torch.zeros(4, **i32))
    with pytest.raises(MI355AttnError, match="bidir_lens"):
        c.run(bidir_lens=torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(MI355AttnError, match="rows for"):
        c.run(decode=True)
    with pytest.raises(MI355AttnError, match="dtype"):
        c.run(q=c.q.reshape(5, -1).to(DEV).half())
    with pytest.raises(MI355AttnError, match="out"):
        c.run(out=torch.empty((5, 255), dtype=BF, device=DEV))
    with pytest.raises(MI355AttnError):
        c.run(softcap=-1.0)
    with pytest.raises(MI355AttnError):
        c.run(window=-2)
    with pytest.raises(MI355AttnError):
        c.run(scale=0.0)
    with pytest.raises(MI355AttnError, match="fit"):
        c.run(window=2 ** 40)
    with pytest.raises(MI355AttnError):
        c.run(softcap=1e300)


def test_two_calls_at_once():
    """Calls on two streams, each over its own workspace, with splits and without: every one gives what it gives alone."""
    cases = [(Case(25, BF, (8, 2, 64), 16, [1500, 40], [1, 1]), dict(decode=True, softcap=30.0)),
             (Case(26, HF, (4, 1, 128), 16, [900, 5], [60, 33]), dict(window=400))]
    alone = [c.run(**kw) for c, kw in cases]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(5):
        for (c, kw), side in zip(cases, sides):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got.append(c.run(**kw))
    torch.cuda.synchronize()
    assert all(torch.equal(o, alone[i % 2]) for i, o in enumerate(got))


def test_one_table_row_for_several_requests():
    """Requests that share a row of the page table: the same tokens, of different lengths."""
    c = Case(27, BF, (4, 2, 64), 16, [200, 200, 200], [1, 1, 1])
    c.rows[1:] = c.rows[0]
    c.len, c.pre = [201, 150, 7], [200, 149, 6]
    c.slots = [c.slots[0][:n] for n in c.len]
    check(c.run(decode=True, softcap=30.0), *c.want(softcap=30.0))
    c.pre, c.ext, c.len, c.cu = [100, 0, 3], [60, 60, 60], [160, 60, 63], [0, 60, 120, 180]
    c.T = 180
    c.q = torch.randn((180, 4, 64), generator=c.g).to(BF)
    c.slots = [([int(c.table[c.rows[0], t // 16]) * 16 + t % 16 for t in range(n)]) for n in c.len]
    check(c.run(slopes=slopes_of(4).to(DEV)), *c.want(slopes=slopes_of(4)))
