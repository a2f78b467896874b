"""Speculative decoding on the harness runner: drafts come from the request's own history, a tree of them is verified in one
forward, and the longest path the model agrees with is kept.

One step, for every request of the batch at once:
    draft       continuations of earlier occurrences of the last tokens, merged into a tree rooted at the token sampled last
    verify      Batch.prepare_for_tree (one metadata launch) and a forward whose attention layers run ops.tree_attn: logits of
                every node
    accept      ops.token_logprobs gives each node's most likely next token and its log probability; from the root, a child whose
                token is its parent's most likely one is accepted
    commit      Batch.commit_tree moves the path's K/V to its positions and gives the other pages back
With greedy sampling the tokens are those of the one-token-at-a-time loop, up to the rounding of the two attention forms.
"""
from __future__ import annotations

from typing import Callable, List, Sequence, Tuple

import torch

import mi355_attn as m

Tree = Tuple[List[int], List[int]]                       # tokens, parents (node 0 is the token sampled last)


def history_tree(history: Sequence[int], nodes: int, depth: int = 6) -> Tree:
    """A draft tree of at most `nodes` tokens for a history that ends with the token sampled last: what followed that token's
    earlier occurrences (the latest first), up to `depth` tokens each; common beginnings share nodes."""
    tokens, parents, children = [history[-1]], [-1], {}
    for at in range(len(history) - 2, -1, -1):
        if len(tokens) >= nodes:
            break
        if history[at] != history[-1]:
            continue
        node = 0
        for tok in history[at + 1:at + 1 + depth]:
            nxt = children.get((node, tok))
            if nxt is None:
                if len(tokens) >= nodes:
                    break
                nxt = children[(node, tok)] = len(tokens)
                tokens.append(tok)
                parents.append(node)
            node = nxt
    return tokens, parents


def accepted_path(tree: Tree, best: Sequence[int]) -> List[int]:
    """Nodes from the root down for as long as a child's token is its parent's most likely next one."""
    tokens, parents = tree
    path, node = [0], 0
    while True:
        nxt = next((j for j in range(node + 1, len(tokens)) if parents[j] == node and tokens[j] == best[node]), None)
        if nxt is None:
            return path
        path.append(nxt)
        node = nxt


@torch.no_grad()
def speculative_decode(runner, next_ids: torch.Tensor, batch, new_tokens: int, nodes: int = 8,
                       draft: Callable[[Sequence[int], int], Tree] = history_tree):
    """Greedy decode of `new_tokens` more tokens per request after a prefill whose sampled ids are `next_ids`.  Returns (ids
    [B][new_tokens], their log probabilities, verification steps taken)."""
    first = next_ids.tolist()
    history = [list(r.origin_input_ids) + [t] for r, t in zip(batch.reqs, first)]
    out: List[List[int]] = [[] for _ in first]
    logprobs: List[List[float]] = [[] for _ in first]
    steps = 0
    while min(len(o) for o in out) < new_tokens:
        # (a request that is done stays in the batch with its last token as a tree of one, of which nothing is kept)
        trees = [draft(h, max(1, min(nodes, new_tokens - len(o)))) for h, o in zip(history, out)]
        batch.prepare_for_tree([t for t, _ in trees], [p for _, p in trees])
        logits, _ = runner.forward(batch)
        top = m.ops.token_logprobs(logits, top_k=1)
        best, lps = top.top_ids[:, 0].tolist(), top.top_logprobs[:, 0].tolist()
        paths, at = [], 0
        for b, tree in enumerate(trees):
            n = len(tree[0])
            path = accepted_path(tree, best[at:at + n]) if len(out[b]) < new_tokens else []
            got = [best[at + node] for node in path]
            history[b] += got
            out[b] += got
            logprobs[b] += [lps[at + node] for node in path]
            paths.append(path)
            at += n
        batch.commit_tree(paths)
        steps += 1
    return [o[:new_tokens] for o in out], [lp[:new_tokens] for lp in logprobs], steps
