"""The operators a serving engine needs around plain paged attention, in their plain form and as the framework offers them.

Three operators, each with the cases it is measured on:

  scored   attention over the paged KV pools whose scores are capped by a tanh, biased by distance (one slope per head) or
           limited by a window, a document mask or a bidirectional prefix - extend and single-token form
  tree     attention of a tree of drafted tokens over the cache: the tree's metadata (ancestor mask, positions, slots, page
           table) and the attention that reads it
  logprobs log probabilities of given tokens, the entropy of the row and its most likely alternatives, from logits

`own` selects which of the two `run` calls.  The plain form is elementary torch in 32 bits, rounded once; `exact` is the
definition in 64 bits, request by request.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ESIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------------ cases
def _scored(name, dtype, B, heads, ps, pre, ext, cap=0.0, alibi=False, window=0, doc=0, bidir=False):
    return {"name": name, "op": "scored", "dtype": dtype, "B": B, "Hq": heads[0], "Hkv": heads[1], "D": heads[2], "ps": ps,
            "pre_lo": pre[0], "pre_hi": pre[1], "ext_lo": ext[0], "ext_hi": ext[1], "cap": cap, "alibi": alibi,
            "window": window, "doc": doc, "bidir": bidir}


def _tree(name, dtype, B, heads, ps, pre, nodes, depth, cap=0.0, alibi=False):
    return {"name": name, "op": "tree", "dtype": dtype, "B": B, "Hq": heads[0], "Hkv": heads[1], "D": heads[2], "ps": ps,
            "pre_lo": pre[0], "pre_hi": pre[1], "ext_lo": nodes[0], "ext_hi": nodes[1], "depth": depth, "cap": cap,
            "alibi": alibi}


def _logprobs(name, dtype, T, V, given, k, temperature):
    return {"name": name, "op": "logprobs", "dtype": dtype, "T": T, "V": V, "given": given, "k": k, "temperature": temperature}


def listed():
    return [
        # one request of a few hundred tokens, one step: what a single user waits for (latency)
        _scored("decode_cap_single", "bf16", 1, (32, 8, 128), 16, (640, 640), (1, 1), cap=50.0),
        # a ragged serving batch's decode step, the lengths of the headline decode benchmark, scores capped
        _scored("decode_cap_ragged", "bf16", 64, (32, 8, 64), 16, (63, 2047), (1, 1), cap=50.0),
        # the per-rank step of a long-context batch under tensor parallelism, biased by distance, half precision
        _scored("decode_bias_long", "fp16", 16, (8, 1, 128), 16, (20000, 32767), (1, 1), alibi=True),
        # new turns over a shared-prefix-sized cached history, capped scores in every layer
        _scored("extend_cap_turns", "bf16", 16, (32, 8, 128), 16, (1024, 1024), (384, 640), cap=30.0),
        # documents packed into long prompts, each attending itself only
        _scored("extend_documents", "bf16", 2, (32, 8, 64), 16, (0, 0), (7001, 8192), doc=700),
        # odd everything: pages of one token, three query heads per kv head, a bidirectional prompt prefix and a bias
        _scored("extend_prefix_odd", "fp16", 5, (6, 2, 64), 1, (0, 333), (77, 411), alibi=True, bidir=True),
        # a sliding window over long histories, short turns: most of the cache must not be read
        _scored("extend_window_short", "bf16", 8, (32, 8, 128), 16, (6000, 16000), (5, 40), window=4096),
        # one request verifying a small draft: latency
        _tree("tree_single", "bf16", 1, (32, 8, 128), 16, (700, 700), (8, 8), 4),
        # a serving batch verifying drafts of mixed sizes
        _tree("tree_batch", "bf16", 16, (32, 8, 128), 16, (500, 4000), (17, 48), 8),
        # large trees over long histories on one rank of a tensor-parallel group, capped
        _tree("tree_long_cap", "bf16", 4, (8, 1, 128), 16, (20001, 32000), (64, 64), 10, cap=50.0),
        # the sampled tokens of a decode step's batch
        _logprobs("logprobs_step", "bf16", 64, 128256, 1, 20, 1.0),
        # every prompt token scored (evaluation), logits kept in 32 bits
        _logprobs("logprobs_prompt", "fp32", 1500, 128256, 1, 5, 0.7),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "fp16"])
    ps = rng.choice([1, 3, 16, 16, 64])
    cap = rng.choice([0.0, 30.0, 50.0])
    alibi = rng.random() < 0.4
    kind = rng.choice(["decode", "extend", "tree", "logprobs"])
    if kind == "logprobs":
        V = _log(rng, 100, 130000)
        T = min(_log(rng, 1, 2000), max(1, 180_000_000 // V))
        return {k: v for k, v in _logprobs("", rng.choice(["bf16", "fp16", "fp32"]), T, V, rng.choice([1, 1, 4]),
                                           min(V, rng.choice([0, 1, 5, 20, 64])), rng.choice([1.0, 0.7, 1.3])).items() if k != "name"}
    D = rng.choice([64, 128])
    Hkv = rng.choice([1, 2, 8])
    Hq = Hkv * rng.choice([1, 2, 3, 4, 5, 8])
    if kind == "decode":
        B = _log(rng, 1, 128)
        hi = _log(rng, 2, max(3, min(32768, 300000 // B)))
        c = _scored("", dtype, B, (Hq, Hkv, D), ps, (rng.randint(0, hi - 1), hi), (1, 1), cap, alibi, rng.choice([0, 0, 1000]))
    elif kind == "extend":
        B = _log(rng, 1, 24)
        ext = _log(rng, 2, max(3, 8192 // B))
        pre = rng.choice([0, _log(rng, 1, max(2, 16384 // B))])
        c = _scored("", dtype, B, (Hq, Hkv, D), ps, (rng.randint(0, pre), pre), (rng.randint(1, ext), ext), cap, alibi,
                    rng.choice([0, 0, 500]), rng.choice([0, 0, 150]), rng.random() < 0.3)
    else:
        B = _log(rng, 1, 32)
        pre = _log(rng, 1, max(2, min(32768, 120000 // B)))
        n = _log(rng, 2, 100)
        c = _tree("", dtype, B, (Hq, Hkv, D), ps, (rng.randint(0, pre), pre), (rng.randint(1, n), n), rng.randint(1, 12), cap, alibi)
    while work(c)["flops"] > 1.7e11 or work(c)["bytes"] > 7.5e8:                     # no more than the largest listed case
        c["pre_lo"], c["pre_hi"] = c["pre_lo"] * 3 // 4, c["pre_hi"] * 3 // 4
        c["ext_lo"], c["ext_hi"] = max(1, c["ext_lo"] * 3 // 4), max(1, c["ext_hi"] * 3 // 4)
    return {k: v for k, v in c.items() if k != "name"}


# ------------------------------------------------------------------------------------------------ layout of a case
def _spread(lo, hi, n, phase):
    """n whole numbers spread evenly over [lo, hi] in a scrambled order; the first is hi."""
    at = (1.0 - (np.arange(n) * 0.6180339887498949 + phase) % 1.0)
    at[0] = 1.0
    return np.minimum(hi, lo + np.floor(at * (hi - lo + 1))).astype(np.int64)


def _layout(c):
    """Lengths and masks: they follow from the case alone, values and pages from the seed."""
    pre, ext = _spread(c["pre_lo"], c["pre_hi"], c["B"], 0.0), _spread(c["ext_lo"], c["ext_hi"], c["B"], 0.37)
    cu = np.concatenate([[0], np.cumsum(ext)])
    pos = np.concatenate([p + np.arange(e) for p, e in zip(pre, ext)])
    L = {"pre": pre, "ext": ext, "len": pre + ext, "cu": cu, "pos": pos, "req": np.repeat(np.arange(c["B"]), ext)}
    lo, hi = np.zeros_like(pos), pos + 1
    if c.get("doc"):
        # documents of a few hundred to a thousand tokens: boundaries at uneven steps of every sequence
        edges = np.cumsum(_spread(c["doc"] // 3, 2 * c["doc"], 2 + int(6 * L["len"].max() / c["doc"]), 0.11))
        edges = np.concatenate([[0], edges])
        L["doc_start"] = edges[np.searchsorted(edges, pos, side="right") - 1]
        lo = np.maximum(lo, L["doc_start"])
    if c.get("window"):
        lo = np.maximum(lo, pos - c["window"] + 1)
    if c.get("bidir"):
        L["bidir"] = pre + (ext + 1) // 2
        hi = np.maximum(hi, L["bidir"][L["req"]])
    L["lo"], L["hi"] = lo, hi
    return L


def work(case):
    if case["op"] == "logprobs":
        n = case["T"] * case["V"]
        return {"bytes": n * ESIZE[case["dtype"]] + case["T"] * (case["given"] * 12 + 4 + case["k"] * 12), "flops": 6 * n}
    L = _layout(case)
    width = case["D"] * ESIZE[case["dtype"]]
    if case["op"] == "tree":
        keys, pairs = int(L["len"].sum()), int((L["ext"] * L["pre"]).sum() + L["ext"].sum() * min(case["depth"], 8))
    else:
        first = [int(L["lo"][a:b].min()) for a, b in zip(L["cu"][:-1], L["cu"][1:])]
        last = [int(L["hi"][a:b].max()) for a, b in zip(L["cu"][:-1], L["cu"][1:])]
        keys, pairs = sum(b - a for a, b in zip(first, last)), int((L["hi"] - L["lo"]).sum())
    return {"bytes": 2 * keys * case["Hkv"] * width + 2 * int(L["cu"][-1]) * case["Hq"] * width,
            "flops": 4 * pairs * case["Hq"] * case["D"]}


# ------------------------------------------------------------------------------------------------ inputs
def _drafts(rng, n, depth):
    """Parents of n drafted nodes in topological order (the first is the last accepted token, the tree's root)."""
    parents, level = [-1], [0]
    for j in range(1, n):
        a = rng.randrange(max(0, j - 9), j)
        if level[a] + 1 > depth:
            a = 0
        parents.append(a)
        level.append(level[a] + 1)
    return parents


def _slopes(heads):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)], dtype=torch.float32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "logprobs":
        T, V = case["T"], case["V"]
        x = torch.randn((T, V), generator=g, device=DEV, dtype=torch.float32).mul_(3.0)
        x.add_(torch.randn((T, 1), generator=g, device=DEV))
        return {"case": case, "logits": x.to(dtype),
                "tokens": torch.randint(0, V, (T, case["given"]), generator=g, device=DEV)}
    L, ps, B = _layout(case), case["ps"], case["B"]
    Hq, Hkv, D, T = case["Hq"], case["Hkv"], case["D"], int(L["cu"][-1])
    pages = -(-L["len"] // ps)
    width = int(pages.max()) + 1
    total = int(pages.sum())
    order = torch.randperm(total + 3, generator=g, device=DEV).to(torch.int32)
    rows = torch.randperm(B + 2, generator=g, device=DEV)[:B]
    dev = lambda a, t: torch.as_tensor(np.ascontiguousarray(a), dtype=t).to(DEV)  # noqa: E731
    req = dev(np.repeat(np.arange(B), pages), torch.int64)
    col = dev(np.concatenate([np.arange(n) for n in pages]), torch.int64)
    table = torch.zeros((B + 2, width), dtype=torch.int32, device=DEV)
    row = Hkv * D
    pitch = row + (64 if row >= 512 and row % 128 == 0 else 0)          # the pools' row padding (KVCache)
    pools = torch.randn((2, (total + 3) * ps, pitch), generator=g, device=DEV, dtype=dtype)
    s = {"case": case, "q": torch.randn((T, Hq * D), generator=g, device=DEV).mul_(3.0).to(dtype),
         "k": pools[0, :, :row].unflatten(1, (Hkv, D)), "v": pools[1, :, :row].unflatten(1, (Hkv, D)), "table": table,
         "rows": rows, "pre": dev(L["pre"], torch.int64), "len": dev(L["len"], torch.int64), "cu": dev(L["cu"], torch.int32),
         "max_len": int(L["len"].max()), "max_ext": int(L["ext"].max()), "slopes": _slopes(Hq) if case["alibi"] else None}
    if case["op"] == "scored":
        table[rows[req], col] = order[:total]
        s["doc_start"] = dev(L["doc_start"], torch.int32) if case["doc"] else None
        s["bidir"] = dev(L["bidir"], torch.int32) if case["bidir"] else None
        return s
    # a tree's nodes take new pages behind the ones the prefix has: the metadata call enters them into the table
    held = -(-L["pre"] // ps)
    old = dev(np.concatenate([np.arange(n) for n in pages]) < np.repeat(held, pages), torch.bool)
    table[rows[req[old]], col[old]] = order[:total][old]
    s["new_pages"] = order[:total][~old].contiguous()
    s["new_off"] = dev(np.concatenate([[0], np.cumsum(pages - held)]), torch.int32)
    rng = random.Random(seed)
    s["parents"] = dev(np.concatenate([_drafts(rng, int(n), case["depth"]) for n in L["ext"]]), torch.int32)
    return s


# ------------------------------------------------------------------------------------------------ the framework's operators
def _ops():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-sglang_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from mi355_attn import ops
    return ops


def _run_own(s):
    ops, c = _ops(), s["case"]
    if c["op"] == "logprobs":
        r = ops.token_logprobs(s["logits"], s["tokens"], top_k=c["k"], temperature=c["temperature"])
        return {"logprobs": r.logprobs, "entropy": r.entropy, "top_logprobs": r.top_logprobs, "top_ids": r.top_ids}
    if c["op"] == "scored":
        form = {} if c["ext_hi"] == 1 else {"prefix_lens": s["pre"], "cu_q": s["cu"], "max_extend_len": s["max_ext"]}
        return {"out": ops.scored_attn(s["q"], s["k"], s["v"], s["table"], s["rows"], s["len"], c["ps"], c["Hq"], s["max_len"],
                                       softcap=c["cap"], slopes=s["slopes"], window=c["window"], doc_starts=s["doc_start"],
                                       bidir_lens=s["bidir"], **form)}
    plan = ops.tree_prepare(s["table"], s["rows"], s["pre"], s["parents"], s["cu"], c["ps"], s["max_ext"],
                            new_pages=s["new_pages"], new_page_off=s["new_off"])
    out = ops.tree_attn(s["q"], s["k"], s["v"], s["table"], s["rows"], s["pre"], plan, c["ps"], c["Hq"], s["max_len"],
                        softcap=c["cap"], slopes=s["slopes"])
    return {"out": out, "positions": plan.positions, "slots": plan.out_cache_loc, "table": s["table"]}


# ------------------------------------------------------------------------------------------------ the plain form
def _rows_of(s):
    """Request and place inside the request of every query row."""
    n = s["cu"].long()
    req = torch.repeat_interleave(torch.arange(s["case"]["B"], device=DEV), n[1:] - n[:-1], output_size=s["q"].shape[0])
    return req, torch.arange(s["q"].shape[0], device=DEV) - n[req]


def _slots_of(s, req, pos):
    ps = s["case"]["ps"]
    col = torch.clamp(pos // ps, max=s["table"].shape[1] - 1)
    return s["table"][s["rows"][req], col].long() * ps + pos % ps


def _attend(s, visible, q_pos, k_pos, req, place):
    """softmax(f(q k^T)) v over padded requests in 32 bits; visible [B, E, L], positions [B, E] and [B, L]."""
    c = s["case"]
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    G, E, n = Hq // Hkv, visible.shape[1], visible.shape[2]
    keys = torch.arange(n, device=DEV)
    slots = _slots_of(s, torch.arange(B, device=DEV)[:, None], torch.minimum(keys[None, :], s["len"][:, None] - 1))
    k = s["k"][slots].float().permute(0, 2, 3, 1).contiguous()                      # [B, Hkv, D, n]
    v = s["v"][slots].float().permute(0, 2, 1, 3).contiguous()                      # [B, Hkv, n, D]
    q = torch.zeros((B, E, Hkv, G, D), device=DEV)
    q[req, place] = s["q"].float().view(-1, Hkv, G, D)
    scores = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * E, D), k).mul_(D ** -0.5).view(B, Hkv, G, E, n)
    if c["cap"]:
        scores = scores.div_(c["cap"]).tanh_().mul_(c["cap"])
    if c["alibi"]:
        away = (q_pos[:, :, None] - k_pos[:, None, :]).abs().float()
        scores = scores.sub_(s["slopes"].view(1, Hkv, G, 1, 1) * away[:, None, None])
    scores = scores.masked_fill_(~visible[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, Hkv, G * E, n), v).view(B, Hkv, G, E, D) / torch.where(total > 0, total, torch.ones_like(total))
    return out.permute(0, 3, 1, 2, 4)[req, place].reshape(-1, Hq * D).to(s["q"].dtype)


def _plain_scored(s):
    c = s["case"]
    req, place = _rows_of(s)
    keys = torch.arange(s["max_len"], device=DEV)
    pos = s["pre"][:, None] + torch.arange(s["max_ext"], device=DEV)[None, :]        # [B, E]
    lo, hi = torch.zeros_like(pos), pos + 1
    if c["doc"]:
        lo[req, place] = s["doc_start"].long()
    if c["window"]:
        lo = torch.maximum(lo, pos - c["window"] + 1)
    if c["bidir"]:
        hi = torch.maximum(hi, s["bidir"].long()[:, None])
    visible = (keys >= lo[:, :, None]) & (keys < torch.minimum(hi, s["len"][:, None])[:, :, None])
    return {"out": _attend(s, visible, pos, keys[None, :].expand(c["B"], -1), req, place)}


def _plain_tree(s):
    c = s["case"]
    B, N = c["B"], s["max_ext"]
    off = s["new_off"].long()
    owner = torch.repeat_interleave(torch.arange(B, device=DEV), off[1:] - off[:-1], output_size=s["new_pages"].shape[0])
    first = (s["pre"] + c["ps"] - 1) // c["ps"]
    column = first[owner] + torch.arange(owner.shape[0], device=DEV) - off[owner]
    s["table"][s["rows"][owner], column] = s["new_pages"]
    req, place = _rows_of(s)
    child = s["parents"] >= 0
    step = torch.zeros((B, N, N), device=DEV)
    step[req[child], place[child], s["parents"][child].long()] = 1.0
    step.diagonal(dim1=1, dim2=2).fill_(1.0)
    above = torch.linalg.matrix_power(step, max(1, c["depth"])) > 0                 # [B, node, ancestor or itself]
    level = above.sum(-1) - 1
    keys = torch.arange(s["max_len"], device=DEV)[None, :].expand(B, -1)
    node = keys - s["pre"][:, None]                                                  # [B, L]: which node of the tree, or < 0
    at = node.clamp(0, N - 1)
    tail = (node >= 0) & (keys < s["len"][:, None])
    hit = torch.gather(above, 2, at[:, None, :].expand(-1, N, -1))
    visible = (node < 0)[:, None, :] | (tail[:, None, :] & hit)
    k_pos = torch.where(node < 0, keys, s["pre"][:, None] + torch.gather(level, 1, at))
    q_pos = s["pre"][:, None] + level
    out = _attend(s, visible, q_pos, k_pos, req, place)
    return {"out": out, "positions": q_pos[req, place], "slots": _slots_of(s, req, s["pre"][req] + place), "table": s["table"]}


def _plain_logprobs(s):
    c = s["case"]
    raw = s["logits"].float() + 0.0
    top = raw.amax(-1, keepdim=True)
    x = (raw - top) / c["temperature"]
    e = x.exp()
    total = e.sum(-1, keepdim=True)
    logz = total.log()
    entropy = (logz - (e * x).sum(-1, keepdim=True) / total).squeeze(-1)
    # the order of 32-bit floats as whole numbers, the lower index first among equals
    bits = raw.view(torch.int32).long()
    order = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF)
    key = order * (1 << 32) + (0xFFFFFFFF - torch.arange(c["V"], device=DEV))
    ids = 0xFFFFFFFF - (torch.topk(key, c["k"], dim=-1).values & 0xFFFFFFFF)
    return {"logprobs": torch.gather(x, 1, s["tokens"]) - logz, "entropy": entropy,
            "top_logprobs": torch.gather(x, 1, ids) - logz, "top_ids": ids}


def run(state):
    if own:
        return _run_own(state)
    return {"scored": _plain_scored, "tree": _plain_tree, "logprobs": _plain_logprobs}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def _exact_logprobs(s):
    c = s["case"]
    got = {"logprobs": [], "entropy": [], "top_logprobs": [], "top_ids": None}
    for a in range(0, c["T"], 128):
        raw = s["logits"][a:a + 128].double()
        lp = torch.log_softmax(raw / c["temperature"], -1)
        got["logprobs"].append(torch.take_along_dim(lp, s["tokens"][a:a + 128], 1))
        got["entropy"].append(-(lp.exp() * lp).sum(-1))
        got["top_logprobs"].append(torch.sort(lp, dim=-1, descending=True).values[:, :c["k"]])
    return {k: v if v is None else torch.cat(v) for k, v in got.items()}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(s)
    L, ps, Hkv, D = _layout(case), case["ps"], case["Hkv"], case["D"]
    G = case["Hq"] // Hkv
    T = int(L["cu"][-1])
    out = torch.zeros((T, Hkv, G, D), dtype=torch.float64, device=DEV)
    table, parents = s["table"].cpu().numpy().copy(), None
    if case["op"] == "tree":
        off, fresh, parents = s["new_off"].tolist(), s["new_pages"].cpu().numpy(), s["parents"].tolist()
        for b, r in enumerate(s["rows"].tolist()):
            c0 = -(-int(L["pre"][b]) // ps)
            table[r, c0:c0 + off[b + 1] - off[b]] = fresh[off[b]:off[b + 1]]
    for b, r in enumerate(s["rows"].tolist()):
        P, E, n = int(L["pre"][b]), int(L["ext"][b]), int(L["len"][b])
        a = int(L["cu"][b])
        seen = np.zeros((E, n), dtype=bool)
        key_pos, query_pos = np.arange(n), P + np.arange(E)
        if parents is None:
            for j in range(E):
                seen[j, L["lo"][a + j]:min(n, L["hi"][a + j])] = True
        else:
            for j in range(E):
                up = parents[a + j]
                seen[j, :P], seen[j, P + j] = True, True
                query_pos[j] = P
                if up >= 0:
                    seen[j, P:] |= seen[up, P:]
                    query_pos[j] = query_pos[up] + 1
            key_pos[P:] = query_pos
        token = np.arange(n)
        slot = torch.from_numpy(table[r, token // ps].astype(np.int64) * ps + token % ps).to(DEV)
        hide = torch.from_numpy(~seen).to(DEV)
        away = torch.from_numpy(np.abs(query_pos[:, None] - key_pos[None, :])).to(DEV)
        for h in range(Hkv):
            k, v = s["k"][slot, h].double(), s["v"][slot, h].double()
            for i in range(G):
                head = h * G + i
                x = s["q"][a:a + E, head * D:(head + 1) * D].double() @ k.t() / math.sqrt(D)
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                if case["alibi"]:
                    x = x - float(s["slopes"][head]) * away
                w = torch.softmax(x.masked_fill(hide, -math.inf), -1)
                out[a:a + E, h, i] = torch.nan_to_num(w) @ v
    out = out.reshape(T, case["Hq"] * D)
    return {"out": out} if parents is None else {"out": out, "positions": None, "slots": None, "table": None}
