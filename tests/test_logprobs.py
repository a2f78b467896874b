"""m355_token_logprobs on the GPU against log-softmax in 64 bits; ids exactly, values to oracle/scored_ref.py's bound."""
import pytest
import torch

from oracle.scored_ref import logprobs_bound, logprobs_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check(x, tokens, k, temp=1.0, **kw):
    from mi355_attn import ops
    r = ops.token_logprobs(x if x.is_cuda else x.to(DEV), None if tokens is None else tokens.to(DEV), top_k=k, temperature=temp, **kw)
    x = x.cpu()
    lp, ent, ids = logprobs_ref(x, tokens, k, temp)
    top = x.double().amax(-1, keepdim=True)
    base = logprobs_bound(x, temp)

    def near(got, want, at):
        # (x - max) / temperature: one rounding of the difference, of 1 / temperature, of the product; the last subtraction one more
        d = ((x.double().gather(1, at) - top) / temp).abs().nan_to_num(posinf=0.0)
        tol = base + 2.0 ** -24 * (4 * d + 2 * want.abs().nan_to_num(posinf=0.0))
        got = got.double().cpu()
        same = torch.isfinite(want)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(torch.isinf(got), torch.isinf(want))
        assert bool(((got - want).abs() <= tol)[same].all()), float(((got - want).abs() - tol)[same].max())

    assert torch.equal(r.top_ids.cpu(), ids)
    near(r.top_logprobs, lp.gather(1, ids), ids)
    if tokens is not None:
        at = tokens.view(len(x), -1)
        ok = (at >= 0) & (at < x.shape[1])
        want = torch.where(ok, lp.gather(1, at.clamp(0, x.shape[1] - 1)), torch.full((1,), float("-inf"), dtype=torch.float64))
        near(r.logprobs.view(len(x), -1), want, at.clamp(0, x.shape[1] - 1))
        assert r.logprobs.shape == tokens.shape
    # entropy = log S - A / S: the bound of log S, and A / S moves by the same relative error and its terms' rounding
    got = r.entropy.double().cpu()
    assert torch.equal(got.isnan(), ent.isnan())
    fine = ~ent.isnan()
    slack = base * (2 + 2 * ent.abs()) + 2.0 ** -22 * (1 + ent.abs())
    assert bool(((got - ent).abs() <= slack)[fine].all()), float(((got - ent).abs() - slack)[fine].max())
    return r


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,V,k,given", [(1, 1, 1, 1), (3, 2, 2, 2), (5, 63, 5, 1), (7, 1000, 64, 3), (2, 50001, 20, 1), (1, 128256, 20, 1),
                                         (33, 8193, 7, 0), (300, 513, 1, 1), (4, 32000, 0, 5)])
def test_random_rows(dtype, T, V, k, given):
    g = torch.Generator().manual_seed(T * V)
    x = (torch.randn((T, V), generator=g) * 3 + torch.randn((T, 1), generator=g) * 5).to(dtype)
    tokens = torch.randint(0, V, (T, given), generator=g) if given else None
    check(x, tokens, k, 1.0)
    check(x, tokens[:, 0].contiguous() if given else None, k, 0.6)


@pytest.mark.parametrize("V", [257, 40000])
def test_ties_go_to_the_lower_id(V):
    check(torch.zeros((3, V)), torch.zeros(3, dtype=torch.int64), 64)
    x = torch.randint(-2, 3, (4, V), generator=torch.Generator().manual_seed(V)).bfloat16()
    x[0, ::2] = -0.0
    check(x, torch.full((4,), V - 1), 50)


@pytest.mark.parametrize("V", [300, 33000, 128256])
@pytest.mark.parametrize("kind", ["rising", "falling", "spikes-at-the-end", "one-block"])
def test_adversarial_orders(V, kind):
    x = torch.arange(V, dtype=torch.float32) / V * 20
    if kind == "falling":
        x = x.flip(0)
    elif kind == "spikes-at-the-end":
        x = torch.zeros(V)
        x[-70:] = torch.arange(70.0)
    elif kind == "one-block":
        x = torch.zeros(V)
        x[100:180] = 5 + torch.arange(80.0) % 7
    check(torch.stack([x, x * 0.5]), torch.tensor([V - 1, 0]), 64)


def test_masked_vocabularies_and_rows_without_a_distribution():
    inf = float("inf")
    g = torch.Generator().manual_seed(1)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = torch.randn((8, 9001), generator=g).to(dtype)
        x[0, 1:] = -inf                                                     # one token left
        x[1, 5000:] = -inf
        x[2, 7:] = torch.finfo(dtype).min                                   # masks of the type's lowest value
        x[3, :] = torch.finfo(dtype).min                                    # ... everywhere: uniform
        x[4, 77] = float("nan")
        x[5, :] = -inf
        x[6, 3] = inf
        check(x, torch.tensor([[0, 5], [6000, 1], [3, 8], [0, 9000], [0, 77], [0, 1], [3, 4], [-1, 9001]]), 6)


def test_rows_of_nan():
    x = torch.randn((4, 20001), generator=torch.Generator().manual_seed(9))
    x[0, :] = float("nan")
    x[1, ::2] = float("nan")
    x[2, -3:] = float("nan")
    x[3, 100] = -float("nan")
    check(x, torch.tensor([0, 1, 2, 3]), 40)


def test_tokens_outside_the_vocabulary():
    x = torch.randn((3, 100), generator=torch.Generator().manual_seed(2))
    check(x, torch.tensor([-1, 100, 2 ** 40]), 0)


def test_ids_outside_where_a_row_has_no_distribution():
    """The row's NaN comes first, whatever the id."""
    from mi355_attn import ops
    x = torch.zeros((4, 50))
    x[0], x[1, 7], x[2, 3] = float("-inf"), float("nan"), float("inf")
    r = ops.token_logprobs(x.to(DEV), torch.tensor([[50, 1], [-1, 7], [2 ** 40, 3], [50, 0]], device=DEV), top_k=2)
    assert r.logprobs[:3].isnan().all() and r.entropy[:3].isnan().all()
    assert r.logprobs[3, 0] == float("-inf") and torch.isfinite(r.logprobs[3, 1])


def test_rows_of_any_alignment():
    g = torch.Generator().manual_seed(3)
    for dtype in (torch.bfloat16, torch.float32):
        wide = torch.full((9, 5003), 100.0, dtype=dtype, device=DEV)         # neighbours larger than every logit
        for off in (0, 1, 3, 7):
            x = torch.randn((9, 4990), generator=g).to(dtype)
            wide.fill_(100.0)
            wide[:, off:off + 4990] = x.to(DEV)
            check(wide[:, off:off + 4990], torch.randint(0, 4990, (9,), generator=g), 9)


def test_temperature_extremes():
    x = torch.randn((4, 3001), generator=torch.Generator().manual_seed(4)).bfloat16()
    check(x, torch.zeros(4, dtype=torch.int64), 3, 0.01)
    check(x, torch.zeros(4, dtype=torch.int64), 3, 100.0)


def test_deterministic_and_replayable():
    from mi355_attn import ops
    x = torch.randn((6, 60001), device=DEV).bfloat16()
    tok = torch.randint(0, 60001, (6,), device=DEV)
    call = lambda: ops.token_logprobs(x, tok, top_k=20)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for step in range(4):
        x.copy_(torch.randn((6, 60001), device=DEV).bfloat16())
        a, b = call(), call()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for u, v, w in zip(a, b, held):
            assert torch.equal(u, v) and torch.equal(u, w)


def test_empty_and_refusals():
    from mi355_attn import ops
    from mi355_attn._lib import MI355AttnError
    r = ops.token_logprobs(torch.zeros((0, 10), device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV), top_k=2)
    assert r.entropy.shape == (0,) and r.top_ids.shape == (0, 2)
    x = torch.zeros((2, 10), device=DEV)
    for bad in (dict(top_k=11), dict(top_k=-1), dict(temperature=0.0), dict(temperature=float("nan")),
                dict(tokens=torch.zeros(2, dtype=torch.int32, device=DEV)), dict(tokens=torch.zeros(3, dtype=torch.int64, device=DEV))):
        with pytest.raises(MI355AttnError):
            ops.token_logprobs(x, **bad)
    with pytest.raises(MI355AttnError):
        ops.token_logprobs(x.t())
    with pytest.raises(MI355AttnError):
        ops.token_logprobs(x.double())
    with pytest.raises(MI355AttnError, match="supported"):
        ops.token_logprobs(torch.zeros((2, 100), device=DEV), top_k=65)
