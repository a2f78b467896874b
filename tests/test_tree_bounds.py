"""Draft trees whose offsets contradict their rows: which keys count as nodes (csrc/scored_rules.h, built for the host), and on the
GPU that the requests that are in order stay right."""
import ctypes
import os
import random
import subprocess

import pytest
import torch

from test_scored_attn import BF, DEV, Case, check, slopes_of
from test_tree_attn import attn, prepare, trees, want

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHIM = r'''
#include "scored_rules.h"
using namespace m355;
extern "C" void span(int64_t q0, int64_t q1, int64_t P, int64_t T, int64_t tok, int32_t* o) {
    const ReqSpan r = tree_span(q0, q1, P, T, tok); o[0] = r.q0; o[1] = r.E; o[2] = r.P; o[3] = r.L; }
'''


def test_nodes_are_rows_of_the_request(tmp_path):
    """A key at or past P is node key - P wherever positions are read: below E, whatever the offsets say."""
    (tmp_path / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                    "-I", os.path.join(REPO, "mini-sglang_amd", "csrc"), str(tmp_path / "shim.cpp"), "-o", str(tmp_path / "shim.so")], check=True)
    lib = ctypes.CDLL(str(tmp_path / "shim.so"))
    lib.span.argtypes = [ctypes.c_int64] * 5 + [ctypes.c_void_p]
    rng = random.Random(0)
    o = (ctypes.c_int32 * 4)()
    offsets, prefixes = [-2 ** 31, -5, 0, 1, 7, 10, 11, 100, 2 ** 31 - 1], [-2 ** 62, -1, 0, 5, 1000, 2 ** 30, 2 ** 62]
    for _ in range(3000):
        T, tokens = rng.choice([0, 1, 10]), rng.choice([0, 16, 2 ** 30 - 1])
        lib.span(rng.choice(offsets), rng.choice(offsets), rng.choice(prefixes), T, tokens, o)
        q0, E, P, L = o
        assert 0 <= q0 and 0 <= E and q0 + E <= T and -1 <= P and 0 <= L <= tokens
        assert L - 1 - P < max(E, 1), "a key past the last node"
    lib.span(4, 9, 100, 50, 1000, o)                                       # in order: prefix and nodes
    assert list(o) == [4, 5, 100, 105]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(window=3), dict(window=40, slopes=True, softcap=20.0)], ids=lambda k: "-".join(k) or "plain")
def test_offsets_past_the_rows(kw):
    """The last request's offset lies past q: its rows count as far as there are any, the others' results are what they were."""
    c = Case(70, BF, (4, 2, 64), 16, [50, 33, 20], [9, 12, 8])
    parents = trees(71, c.ext)
    plan = prepare(c, parents)
    ref = dict(kw)
    if "slopes" in kw:
        ref["slopes"] = slopes_of(4)
        kw = dict(kw, slopes=ref["slopes"].to(DEV))
    past = plan.cu_q.clone()
    past[3] = 29 + 1000
    mask = plan.mask.clone()
    mask[21:] |= -256                                                      # bits of nodes that no row stands for
    got = attn(c, plan._replace(cu_q=past, mask=mask), **kw)
    check(got, *want(c, parents, **ref))
