"""The index rules of the scored attention (csrc/scored_rules.h), built for the host: visible ranges, tile bits of intervals and
trees, slots of bad pages, rows of inconsistent batches.  And the refusals of the C entry points, which return before any
launch - both on the CPU."""
import ctypes
import os
import random
import subprocess

import pytest

from oracle.scored_ref import ancestors_ref, visible_ref

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SHIM = r'''
#include "scored_rules.h"
using namespace m355;
extern "C" {
void range(int32_t pos, int32_t len, int32_t win, int32_t doc, int32_t bidir, int32_t* lo, int32_t* hi) {
    const KeyRange r = visible_range(pos, len, win, doc, bidir); *lo = r.lo; *hi = r.hi; }
uint32_t rbits(int32_t lo, int32_t hi, int32_t base) { return range_bits(lo, hi, base); }
uint32_t tbits(const uint32_t* m, int32_t w, int32_t P, int32_t hi, int32_t base) { return tree_bits(m, w, P, hi, base); }
int32_t slot(int32_t page, int32_t ps, int32_t off, int64_t S) { return pool_slot(page, ps, off, S); }
void span(int64_t q0, int64_t q1, int64_t P, int64_t L, int64_t T, int64_t tok, int32_t* o) {
    const ReqSpan r = req_span(q0, q1, P, L, T, tok); o[0] = r.q0; o[1] = r.E; o[2] = r.P; o[3] = r.L; }
}
'''


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("rules")
    (d / "shim.cpp").write_text(SHIM)
    so = d / "shim.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                    "-I", os.path.join(REPO, "mini-sglang_amd", "csrc"), str(d / "shim.cpp"), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.rbits.restype = lib.tbits.restype = ctypes.c_uint32
    lib.slot.argtypes = [ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int64]
    lib.span.argtypes = [ctypes.c_int64] * 6 + [ctypes.c_void_p]
    return lib


def test_visible_range_and_tile_bits(rules):
    rng = random.Random(0)
    lo, hi = ctypes.c_int32(), ctypes.c_int32()
    for _ in range(4000):
        length = rng.choice([0, 1, 2, 31, 32, 33, 100, 200])
        pos = rng.randint(-1, length)
        win, doc, bidir = rng.choice([0, 1, 7, 64, 2 ** 31 - 1]), rng.choice([0, 0, 5, 40, 2 ** 30, -3]), rng.choice([0, 0, 50, 2 ** 30])
        rules.range(pos, length, win, doc, bidir, ctypes.byref(lo), ctypes.byref(hi))
        want = visible_ref(pos, length, win, doc, bidir)
        assert list(range(lo.value, hi.value)) == want, (pos, length, win, doc, bidir)
        for base in (0, 32, 64, 192):
            got = rules.rbits(lo.value, hi.value, base)
            assert got == sum(1 << x for x in range(32) if base + x in want)


def test_tree_bits(rules):
    rng = random.Random(1)
    for _ in range(400):
        n, P = rng.choice([1, 2, 31, 32, 33, 64, 70, 130]), rng.choice([0, 1, 5, 31, 32, 40, 63, 64])
        words = -(-n // 32) + rng.choice([0, 0, 1])
        parents = [rng.randint(-1, j - 1) if rng.random() < 0.9 else j + 3 for j in range(n)]
        seen, _ = ancestors_ref(parents)
        for j in rng.sample(range(n), min(n, 6)):
            m = (ctypes.c_uint32 * words)(*[sum(1 << (a & 31) for a in seen[j] if a >> 5 == w) for w in range(words)])
            for base in range(0, P + n + 64, 32):
                want = sum(1 << x for x in range(32) if base + x < P or (base + x - P) in seen[j])
                assert rules.tbits(m, words, P, P + n, base) == want, (n, P, j, base)


def test_bad_pages_stay_inside_the_pool(rules):
    S = 40
    assert [rules.slot(p, 16, o, S) for p, o in ((0, 3), (2, 7), (2, 8), (2 ** 31 - 1, 15), (-1, 0), (-2 ** 31, 5))] == [3, 39, 39, 39, 0, 0]
    assert rules.slot(2 ** 27 - 2, 16, 15, 2 ** 31 - 1) == (2 ** 27 - 2) * 16 + 15


def test_inconsistent_batches_stay_inside_q(rules):
    rng = random.Random(2)
    o = (ctypes.c_int32 * 4)()
    big = [-(2 ** 62), -5, -1, 0, 1, 7, 10, 11, 2 ** 31, 2 ** 62]
    for _ in range(3000):
        T, tokens = rng.choice([0, 1, 10]), rng.choice([0, 16, 2 ** 30 - 1])
        rules.span(rng.choice(big), rng.choice(big), rng.choice(big), rng.choice(big), T, tokens, o)
        q0, E, P, L = o
        assert 0 <= q0 <= T and 0 <= E and q0 + E <= T and -1 <= P < 2 ** 30 and 0 <= L <= tokens


# ------------------------------------------------------------------------------------------------ refusals of the C ABI
A16 = 0x10000                                            # an aligned address that is never followed: the calls return first


def _pack(base, kw):
    from mi355_attn import _lib
    a = {**dict.fromkeys(_lib.SCORED_FIELDS, 0), **base, **kw}
    assert set(a) == set(_lib.SCORED_FIELDS)
    return _lib.SCORED_ARGS.pack(*(a[n] or 0 for n in _lib.SCORED_FIELDS))


_BOTH = dict(q=A16, q_row_stride=512, k_pool=A16, v_pool=A16, pool_rows=64, page_table=A16, pt_row_stride=8, pt_rows=4, pt_cols=8,
             page_table_ids=A16, out=A16, o_row_stride=512, B=2, max_seq_len_hint=100, Hq=8, Hkv=2, D=64, page_size=16, scale=0.125)


def _scored_args(**kw):
    return _pack(dict(_BOTH, seq_lens=A16, T=2, max_extend_len=1), kw)


def _tree_args(**kw):
    return _pack(dict(_BOTH, prefix_lens=A16, cu_q=A16, tree_mask=A16, mask_words=1, T=9, max_extend_len=8), kw)


def test_argument_structure_matches_the_header(tmp_path):
    """The packed bytes are the C structure: same size, every field where the compiler puts it."""
    from mi355_attn import _lib
    (tmp_path / "at.c").write_text('#include <stddef.h>\n#include <stdio.h>\n#include "mi355attn.h"\nint main(void) {\n' +
                                   "".join(f'printf("%zu\\n", offsetof(M355ScoredArgs, {n}));\n' for n in _lib.SCORED_FIELDS) +
                                   'printf("%zu\\n", sizeof(M355ScoredArgs)); return 0; }\n')
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(tmp_path / "at.c"), "-o", str(tmp_path / "at")], check=True)
    where = [int(x) for x in subprocess.run([str(tmp_path / "at")], capture_output=True, text=True, check=True).stdout.split()]
    assert where[-1] == _lib.SCORED_ARGS.size
    n8, n4 = 21, 15
    assert len(_lib.SCORED_FIELDS) == n8 + n4 and where[:-1] == [8 * i for i in range(n8)] + [8 * n8 + 4 * i for i in range(n4)]


INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3
COMMON = [(dict(q=None), INVALID), (dict(out=None), INVALID), (dict(k_pool=A16 + 2), INVALID), (dict(q_row_stride=504), INVALID),
          (dict(o_row_stride=516), INVALID), (dict(pool_row_stride=120), INVALID), (dict(pool_row_stride=132), INVALID), (dict(pool_rows=0), INVALID),
          (dict(pool_rows=2 ** 31), INVALID), (dict(pt_row_stride=7), INVALID), (dict(pt_cols=0), INVALID), (dict(B=-1), INVALID), (dict(T=-1), INVALID),
          (dict(Hq=9), INVALID), (dict(page_size=0), INVALID), (dict(D=96), UNSUPPORTED), (dict(dtype=2), UNSUPPORTED), (dict(scale=0.0), INVALID),
          (dict(scale=float("nan")), INVALID), (dict(softcap=-1.0), INVALID), (dict(softcap=float("inf")), INVALID), (dict(softcap=1e-4), INVALID), (dict(softcap=2000.0), INVALID),
          (dict(softcap=float("nan")), INVALID), (dict(scale=1e20), INVALID), (dict(max_seq_len_hint=0), INVALID),
          (dict(max_extend_len=0, prefix_lens=A16, cu_q=A16), INVALID)]


@pytest.mark.parametrize("bad,code", COMMON + [(dict(window=-1), INVALID), (dict(seq_lens=None), INVALID), (dict(prefix_lens=A16), INVALID),
                                               (dict(cu_q=A16), INVALID), (dict(T=1), INVALID), (dict(tree_mask=A16), INVALID),
                                               (dict(), WORKSPACE)])
def test_scored_attn_refuses(bad, code):
    from mi355_attn import _lib
    assert _lib.load().m355_scored_attn(_scored_args(**bad), None) == code


@pytest.mark.parametrize("bad,code", COMMON + [(dict(prefix_lens=None), INVALID), (dict(cu_q=None), INVALID), (dict(tree_mask=None), INVALID),
                                               (dict(mask_words=0), INVALID), (dict(max_extend_len=33), INVALID), (dict(slopes=A16), INVALID),
                                               (dict(window=5), INVALID), (dict(seq_lens=A16), INVALID), (dict(doc_starts=A16), INVALID),
                                               (dict(), WORKSPACE)])
def test_tree_attn_refuses(bad, code):
    from mi355_attn import _lib
    assert _lib.load().m355_tree_attn(_tree_args(**bad), None) == code


def test_workspace_is_checked():
    from mi355_attn import _lib
    lib = _lib.load()
    need = lib.m355_scored_workspace_bytes(2, 2, 8, 2, 64, 1, 100)
    assert need > 0
    for ws, n in ((A16, need - 1), (A16 + 16, need), (None, need)):
        assert lib.m355_scored_attn(_scored_args(workspace=ws, workspace_bytes=n), None) == WORKSPACE
    assert lib.m355_scored_attn(None, None) == INVALID and lib.m355_tree_attn(None, None) == INVALID
    assert lib.m355_scored_workspace_bytes(0, 2, 8, 2, 64, 1, 100) == 0


def test_empty_calls_do_nothing():
    from mi355_attn import _lib
    lib = _lib.load()
    assert lib.m355_scored_attn(_scored_args(T=0, q=None), None) == 0 and lib.m355_tree_attn(_tree_args(B=0, q=None), None) == 0
    assert lib.m355_tree_prepare(*([None] + [0] * 3 + [None] * 6 + [0, 0, 0, 0, 0, None, 0, None, None, None])) == 0
    assert lib.m355_token_logprobs(None, 0, None, 0, 0, 10, 0, 1.0, None, None, None, None, None, 0, 0, None) == 0


def test_tree_prepare_refuses():
    from mi355_attn import _lib
    base = dict(pt=A16, pts=8, rows=4, cols=8, ids=A16, pre=A16, par=A16, cu=A16, pages=A16, off=A16, count=4, B=2, T=9, nodes=8, ps=16,
                mask=A16, words=1, pos=A16, loc=A16, st=None)
    for bad, code in ((dict(par=None), INVALID), (dict(off=None), INVALID), (dict(count=-1), INVALID), (dict(pts=4), INVALID), (dict(nodes=0), INVALID),
                      (dict(nodes=33), INVALID), (dict(ps=0), INVALID), (dict(nodes=1025, words=33), UNSUPPORTED), (dict(words=33), UNSUPPORTED)):
        assert _lib.load().m355_tree_prepare(*{**base, **bad}.values()) == code, bad


def test_token_logprobs_refuses():
    from mi355_attn import _lib
    base = dict(x=A16, xs=100, tok=A16, given=1, T=4, V=100, k=5, temp=1.0, lp=A16, ent=A16, top=A16, ids=A16, ws=None, wsb=0, dt=0, st=None)
    for bad, code in ((dict(x=None), INVALID), (dict(xs=99), INVALID), (dict(V=0), INVALID), (dict(tok=None), INVALID), (dict(lp=None), INVALID),
                      (dict(ent=None), INVALID), (dict(top=None), INVALID), (dict(k=-1), INVALID), (dict(k=65), UNSUPPORTED),
                      (dict(k=5, V=4, xs=4), UNSUPPORTED), (dict(temp=0.0), INVALID), (dict(temp=float("nan")), INVALID),
                      (dict(temp=1e-38), INVALID), (dict(dt=3), UNSUPPORTED), (dict(x=A16 + 1), INVALID)):
        assert _lib.load().m355_token_logprobs(*{**base, **bad}.values()) == code, bad


def test_python_wrappers_refuse_cpu_tensors():
    import torch
    from mi355_attn import ops
    z = torch.zeros
    with pytest.raises(RuntimeError, match="GPU"):
        ops.scored_attn(z(1, 128), z(4, 2, 64), z(4, 2, 64), z((1, 1), dtype=torch.int32), z(1, dtype=torch.int64), z(1, dtype=torch.int64), 4, 2, 4)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.token_logprobs(z(2, 10))
