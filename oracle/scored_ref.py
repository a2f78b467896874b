"""Attention with modified scores, draft trees and log probabilities in 64 bits, row by row on the CPU: the definition that the
kernels are tested against.  A row works on its visible keys alone, so what masked keys hold cannot matter.

`attend_ref` also returns the bound that its rows' 16-bit results are held to.  With u = eps/2 the relative error of one
rounding of the element type, A = sum_k w_k |v_k| (w: the softmax weights) and delta an error of the scores:
    u |o|       the final rounding
    u A         the weights go into the second matrix product rounded to the element type
    4 delta A   weights and their sum move by e^(2 delta) at most when every score moves by delta
    delta = D 2^-24 max_k sum_i |q_i k_i| scale      (a sum of D products in 32 bits)
          + 8 2^-24 (softcap + max_k |bias_k|)       (a few roundings of the cap's and the bias's terms)
          + 2^-18                                     (exponentials, the running sums over splits)
"""
import numpy as np
import torch


def visible_ref(pos, length, window=0, doc_start=0, bidir=0):
    lo, hi = max(0, doc_start), min(length, max(pos + 1, bidir))
    if window > 0:
        lo = max(lo, pos - window + 1)
    return [k for k in range(lo, hi)]


def ancestors_ref(parents):
    """Per node the set of itself and its ancestors, and its depth."""
    seen, depth = [], []
    for j, up in enumerate(parents):
        ok = 0 <= up < j
        seen.append({j} | (seen[up] if ok else set()))
        depth.append(depth[up] + 1 if ok else 0)
    return seen, depth


def attend_ref(q, k_pool, v_pool, slots, rows, dtype, scale, softcap=0.0, slopes=None):
    """q [E, Hq, D], pools [S, Hkv, D]; slots: slot of every token of the request; rows: per query (visible tokens, their
    positions, own position).  Returns (out, bound), float64 [E, Hq, D]."""
    E, Hq, D = q.shape
    Hkv = k_pool.shape[1]
    G = Hq // Hkv
    u = torch.finfo(dtype).eps / 2
    out, tol = torch.zeros((E, Hq, D), dtype=torch.float64), torch.zeros((E, Hq, D), dtype=torch.float64)
    slots = torch.as_tensor(np.asarray(slots, dtype=np.int64))
    for j, (keys, key_pos, pos) in enumerate(rows):
        if not len(keys):
            continue
        at = slots[torch.as_tensor(np.asarray(keys, dtype=np.int64))]
        away = (torch.as_tensor(np.asarray(key_pos, dtype=np.float64)) - pos).abs()
        k, v = k_pool[at].double(), v_pool[at].double()                       # [n, Hkv, D]
        for h in range(Hq):
            qq, kk, vv = q[j, h].double(), k[:, h // G], v[:, h // G]
            x = kk @ qq * scale
            delta = D * 2.0 ** -24 * float((kk.abs() @ qq.abs()).max()) * scale + 2.0 ** -18
            if softcap:
                x = softcap * torch.tanh(x / softcap)
                delta += 8 * 2.0 ** -24 * softcap
            if slopes is not None:
                bias = float(slopes[h]) * away
                x = x - bias
                delta += 8 * 2.0 ** -24 * float(bias.abs().max())
            w = torch.softmax(x, 0)
            out[j, h] = w @ vv
            tol[j, h] = u * out[j, h].abs() + (u + 4 * delta) * (w @ vv.abs())
    return out, tol


def logprobs_ref(logits, tokens, top_k, temperature):
    """(log p [T, V], entropy [T], top ids [T, k]) in 64 bits; ties to the lower id, NaN first."""
    x = logits.double()
    lp = torch.log_softmax(x / temperature, -1)
    p = lp.exp()
    entropy = -(torch.where(p > 0, p * lp, torch.zeros_like(lp)) + torch.where(p.isnan(), p, torch.zeros_like(p))).sum(-1)
    xs = torch.where(x.isnan(), torch.full_like(x, float("inf")), x).numpy()
    nan = x.isnan().numpy()
    ids = [np.lexsort((np.arange(x.shape[1]), -a, ~n))[:top_k] for a, n in zip(xs, nan)]
    return lp, entropy, torch.from_numpy(np.stack(ids)) if len(ids) else torch.empty((0, top_k), dtype=torch.int64)


def logprobs_bound(logits, temperature):
    """Bound per row on log S, and the rounding of (x - max) / temperature, for any layout in which a thread adds V / 256 terms at most
    one after the other and the partial sums meet pairwise; an exponential is off by its argument's rounding, |d| 2^-23 weighted by
    e^d / S, which is log V 2^-23 at most, and two units of its own.  The kernel's threads add V / 512 at most, fewer where rows are
    split: tests/test_logprobs_sums.py holds it to that."""
    V = logits.shape[1]
    return (V / 256 + 64) * 2.0 ** -24
