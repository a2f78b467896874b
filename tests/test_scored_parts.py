"""The parts that scored attention cuts its keys into: what the device lays out (csrc/scored_rules.h, built for the host) against what
the host reserves, and every part reached exactly once.  On the GPU, batches whose kv heads do not fill whole rounds of 8."""
import ctypes
import os
import random
import subprocess

import pytest
import torch

from test_scored_attn import BF, DEV, HF, Case, check

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# find_share's sums in plain loops: requests with E rows and K keys each
SHIM = r'''
#include "scored_rules.h"
#include <vector>
using namespace m355;
extern "C" int layout(int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t D, int32_t ext, int32_t max_len, const int32_t* E, const int32_t* K,
                      int64_t* reserved, int64_t* wanted, int64_t* bytes) {
    const ScoredCut c = scored_cut(B, T, Hq, Hkv, D, ext, max_len);
    *reserved = c.max_parts; *bytes = c.bytes; *wanted = 0;
    if (!c.slots) return 0;
    const int32_t rb = c.wide ? kWideRows : kFewRows, G = Hq / Hkv;
    float work = 0.f, units = 0.f;
    std::vector<int32_t> blocks(B);
    for (int b = 0; b < B; ++b) {
        blocks[b] = row_blocks(E[b], G, rb, c.blocks);
        work += (float)blocks[b] * (float)K[b];
        units += (float)blocks[b];
    }
    const int32_t size = part_size(work * (float)Hkv, units * (float)Hkv, (float)c.slots, !c.wide);
    for (int b = 0; b < B; ++b) {
        const int32_t n = request_parts(K[b], blocks[b], size, Hkv, !c.wide), items = n * Hkv * blocks[b];
        std::vector<char> seen(items);
        for (int i = 0; i < items; ++i) {
            const PartItem it = part_item(i, blocks[b], n, Hkv);
            if (it.rb < 0 || it.rb >= blocks[b] || it.u < 0 || it.u >= n * Hkv) return 2;
            char& s = seen[it.rb * n * Hkv + it.u];
            if (s) return 3;
            s = 1;
        }
        *wanted += items;
    }
    return *wanted > *reserved;
}
'''


@pytest.fixture(scope="module")
def layout(tmp_path_factory):
    d = tmp_path_factory.mktemp("parts")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                    "-I", os.path.join(REPO, "mini-sglang_amd", "csrc"), str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    lib = ctypes.CDLL(str(d / "shim.so"))

    def call(Hq, Hkv, D, ext, keys, hint_ext=None):
        B, out = len(ext), [ctypes.c_int64() for _ in range(3)]
        code = lib.layout(B, sum(ext), Hq, Hkv, D, hint_ext or max(ext), max(keys), (ctypes.c_int32 * B)(*ext), (ctypes.c_int32 * B)(*keys),
                          *(ctypes.byref(x) for x in out))
        return code, *(x.value for x in out)
    return call


# heads, requests, rows each, tokens each: one part a unit became 4 or 8
ROUNDED = [((40, 10, 128), 20, 64, 1000), ((9, 3, 64), 40, 64, 2000), ((40, 5, 128), 8, 100, 3000), ((28, 7, 128), 14, 64, 1500),
           ((9, 3, 64), 1, 4096, 4096), ((40, 10, 128), 20, 48, 1000)]


@pytest.mark.parametrize("heads,B,rows,tokens", ROUNDED)
def test_parts_of_odd_kv_heads_are_reserved(layout, heads, B, rows, tokens):
    code, reserved, wanted, _ = layout(*heads, [rows] * B, [tokens] * B)
    assert code == 0 and 0 < wanted <= reserved, (wanted, reserved)


@pytest.mark.parametrize("Hkv", range(1, 33))
def test_no_batch_wants_more_parts_than_are_reserved(layout, Hkv):
    """Any batch within its bounds: equal and ragged, extends and single tokens, requests without rows or tokens among them."""
    from mi355_attn import _lib
    rng = random.Random(Hkv)
    split = 0
    for n in range(250):
        G, D, B = rng.choice([1, 2, 3, 4, 5, 7, 8]), rng.choice([64, 128]), int(2 ** rng.uniform(0, 8.01))
        top_e, top_k = int(2 ** rng.uniform(0, 12.5)), int(2 ** rng.uniform(0, 16))
        if n % 2:
            ext, keys = [top_e] * B, [top_e + top_k] * B
        else:
            ext = [rng.choice([0, 1, rng.randint(1, top_e)]) for _ in range(B - 1)] + [top_e]
            keys = [e + rng.choice([0, rng.randint(0, top_k)]) for e in ext]
        code, reserved, wanted, nbytes = layout(G * Hkv, Hkv, D, ext, keys)
        assert code == 0, (code, G, D, ext, keys, wanted, reserved)
        assert nbytes == _lib.load().m355_scored_workspace_bytes(B, sum(ext), G * Hkv, Hkv, D, max(ext), max(keys))
        split += reserved > 0
    assert split > 40


@pytest.mark.parametrize("promised", [1, 4, 40])
def test_rows_past_the_promise_take_no_other_requests_parts(layout, promised):
    """max_extend_len below what some requests bring: those rows may be left out, the parts of all others are still reserved."""
    rng = random.Random(promised)
    for heads in ((8, 1, 64), (8, 2, 128), (9, 3, 64), (32, 8, 128)):
        for _ in range(100):
            B = rng.randint(2, 60)
            ext = [rng.choice([promised, 500]) for _ in range(B)]
            code, reserved, wanted, _ = layout(*heads, ext, [e + rng.randint(100, 3000) for e in ext], hint_ext=promised)
            assert code == 0, (heads, ext, wanted, reserved)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,promised", [((8, 1, 64), 2), ((8, 2, 128), 4), ((4, 1, 64), 40)])
def test_rows_past_the_promise_leave_other_requests_alone(heads, promised):
    """The longest requests stand first: what they bring beyond the promise costs no later request its rows."""
    ext = [200] * 12 + [promised] * 12
    c = Case(63, BF, heads, 16, [700] * 24, ext)
    from mi355_attn import ops
    got = ops.scored_attn(c.q.reshape(c.T, -1).to(DEV), c.pool(c.k), c.pool(c.v), c.table.to(DEV), c.rows.to(DEV), torch.tensor(c.len, device=DEV), 16, c.Hq,
                          max(c.len), prefix_lens=torch.tensor(c.pre, device=DEV), cu_q=torch.tensor(c.cu, dtype=torch.int32, device=DEV),
                          max_extend_len=promised, out=torch.full((c.T, c.Hq * c.D), float("nan"), dtype=BF, device=DEV)).view(c.T, c.Hq, c.D)
    rows = list(range(promised))
    check(got[[c.cu[b] + j for b in range(24) for j in rows]], *c.want(rows=rows))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,B,rows,tokens", ROUNDED)
def test_every_row_of_odd_kv_heads_is_written(heads, B, rows, tokens):
    """A workspace that holds another call's parts, an output of NaN: every row is there, and rows of every block are right."""
    from mi355_attn import ops
    c = Case(60, BF if heads[2] == 128 else HF, heads, 16, [tokens - rows] * B, [rows] * B)
    need = ops.scored_workspace_bytes(B, c.T, c.Hq, c.Hkv, c.D, rows, tokens)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    c.run(q=torch.randn((c.T, c.Hq * c.D), generator=c.g).to(c.dtype).to(DEV), workspace=ws)
    got = c.run(workspace=ws, out=torch.full((c.T, c.Hq * c.D), float("nan"), dtype=c.dtype, device=DEV), softcap=30.0).view(c.T, c.Hq, c.D)
    assert bool(torch.isfinite(got).all())
    per = max(1, 128 // (c.Hq // c.Hkv))                                   # tokens of a row block
    pick = sorted({*range(0, rows, per), rows - 1})
    check(got[[b * rows + j for b in range(B) for j in pick]], *c.want(softcap=30.0, rows=pick))


@pytest.mark.gpu
def test_trees_of_odd_kv_heads():
    from mi355_attn import ops
    from test_tree_attn import prepare, trees, want
    c = Case(61, BF, (40, 10, 128), 16, [952] * 20, [48] * 20)
    parents = trees(62, c.ext)
    plan = prepare(c, parents)
    got = ops.tree_attn(c.q.reshape(c.T, -1).to(DEV), c.pool(c.k), c.pool(c.v), c.table.to(DEV), c.rows.to(DEV), torch.tensor(c.pre, device=DEV),
                        plan, 16, 40, 1000, out=torch.full((c.T, 40 * 128), float("nan"), dtype=BF, device=DEV)).view(c.T, 40, 128)
    assert bool(torch.isfinite(got).all())
    some = [0, 7, 18, 19]                                                  # (the last requests were the ones left out)
    ref, tol = want_of(c, parents, some, want)
    check(got[[c.cu[b] + j for b in some for j in range(48)]], ref, tol)


def want_of(c, parents, requests, want):
    """`want` over some of a batch's requests."""
    import copy
    d = copy.copy(c)
    d.pre, d.slots = [c.pre[b] for b in requests], [c.slots[b] for b in requests]
    at = [c.cu[b] + j for b in requests for j in range(c.ext[b])]
    d.q, d.cu = c.q[at], [sum(c.ext[b] for b in requests[:i]) for i in range(len(requests) + 1)]
    return want(d, [parents[b] for b in requests])
