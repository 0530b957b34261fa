"""The experts' operators as programs run them: on streams of their own, captured and replayed, at sizes whose offsets pass
32 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _parts(T=96, E=8, k=2, D=64, H=96, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return rn(T, E), rn(T, D).to(BF), (0.1 * rn(E, H, D)).to(BF), (0.1 * rn(E, D, H)).to(BF), rn(T, D).to(BF), k


def _step(logits, x, W1, W2, go, k, drop):
    from bitsparse_amd.dropout import dropout
    from bitsparse_amd.experts import expert_combine, expert_linear, plan_experts, route
    leaves = [t.detach().requires_grad_() for t in (logits, x, W1, W2)]
    logits, x, W1, W2 = leaves
    w, ids = route(logits, k)
    plan = plan_experts(ids, W1.shape[0])
    h = torch.relu(expert_linear(x, W1, plan, gather=True))
    out = dropout(expert_combine(expert_linear(h, W2, plan), w, plan), drop)
    return (out, w, ids, *plan, *torch.autograd.grad(out, leaves, go))


@pytest.mark.parametrize("odd", [False, True])
def test_captured_and_replayed(odd):
    """A whole step in one graph: at every replay it routes the logits that are there then, with a mask of its own; replayed
    between eager steps of the same operators."""
    from bitsparse_amd.dropout import Dropout
    parts = _parts(D=61, H=99, T=70) if odd else _parts()
    logits, x, W1, W2, go, k = parts
    state = torch.tensor([3, 0], device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(logits, x, W1, W2, go, k, Dropout(0.2, state))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(logits, x, W1, W2, go, k, Dropout(0.2, state))
    for i in range(5):
        new = _parts(T=70, D=61, H=99, seed=i + 1) if odd else _parts(seed=i + 1)
        for t, n in zip((logits, x, W1, W2, go), new):
            t.copy_(n)
        state.copy_(torch.tensor([3, i]))
        graph.replay()
        torch.cuda.synchronize()
        want = _step(*new, Dropout(0.2, 3, i))
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_streams_at_once():
    """Two streams run steps of their own side by side, with the results of one after the other."""
    from bitsparse_amd.dropout import Dropout
    parts = [_parts(T=500, seed=s) for s in range(2)]
    want = [_step(*p, Dropout(0.3, 1, s)) for s, p in enumerate(parts)]
    streams = [torch.cuda.Stream() for _ in parts]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for s, p in enumerate(parts):
            with torch.cuda.stream(streams[s]):
                got[s].append(_step(*p, Dropout(0.3, 1, s)))
    torch.cuda.synchronize()
    for s in range(2):
        for g in got[s]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[s]))


def test_results_past_32_bits():
    """y and dx of more than 2^31 elements: rows at the start, in the middle and at the end."""
    from bitsparse_amd.experts import expert_combine, expert_linear, plan_experts
    T, E, D, N = 70000, 3, 64, 32768
    ids = (torch.arange(T, device="cuda") % E).int()[:, None].contiguous()
    plan = plan_experts(ids, E)
    x = torch.randn(T, D, device="cuda").to(BF)
    W = torch.randn(E, N, D, device="cuda").to(BF)
    y = expert_linear(x, W, plan, gather=True)
    assert y.numel() > 2 ** 31
    rows = torch.tensor([0, 1, 23333, 23334, 46666, 65535, 65536, 69998, 69999], device="cuda")
    token = plan.order[rows].long()
    want = torch.stack([x[t].double() @ W[ids[t, 0]].double().T for t in token])
    mag = torch.stack([x[t].double().abs() @ W[ids[t, 0]].double().abs().T for t in token])
    assert ((y[rows].double() - want).abs() <= 2.0 ** -8 * want.abs() * 1.02 + (D + 4) * 2.0 ** -24 * mag).all()
    # and the sum over one choice, whose offsets are y's
    w = torch.rand(T, 1, device="cuda")
    out = expert_combine(y, w, plan)
    want = w[token].double() * y[rows].double()
    assert ((out[token].double() - want).abs() <= 2.0 ** -8 * want.abs() * 1.02 + 2.0 ** -23 * want.abs()).all()


def test_gathered_tokens_past_4_gib():
    """Tokens that span 4 GiB: their rows are written out before the product; forward and weight gradient."""
    from bitsparse_amd.experts import expert_linear, plan_experts
    T, E, D, N = 140000, 2, 16384, 16
    ids = torch.full((T, 1), -1, device="cuda", dtype=torch.int32)
    used = torch.tensor([0, 7, 65536, 131072, 131073, 139999], device="cuda")       # padding but for a few
    ids[used, 0] = torch.tensor([0, 1, 0, 1, 1, 0], device="cuda", dtype=torch.int32)
    plan = plan_experts(ids, E)
    x = torch.zeros(T, D, device="cuda", dtype=BF)
    x[used] = torch.randn(len(used), D, device="cuda").to(BF)
    W = torch.randn(E, N, D, device="cuda").to(BF).requires_grad_()
    assert x.numel() * 2 > 2 ** 32
    y = expert_linear(x, W, plan, gather=True)
    token = plan.order[:6].long()
    want = torch.stack([x[t].double() @ W[ids[t, 0]].detach().double().T for t in token])
    mag = torch.stack([x[t].double().abs() @ W[ids[t, 0]].detach().double().abs().T for t in token])
    tol = lambda v, m, n: 2.0 ** -8 * v.abs() * 1.02 + (n + 4) * 2.0 ** -24 * m  # noqa: E731
    assert ((y[:6].double() - want).abs() <= tol(want, mag, D)).all() and (y[6:] == 0).all()
    dy = torch.randn(T, N, device="cuda").to(BF)
    dW, = torch.autograd.grad(y, W, dy)
    for e in range(E):
        r = [i for i in range(6) if ids[token[i], 0] == e]
        a, b = dy[r].double(), x[token[r]].double()
        assert ((dW[e].double() - a.T @ b).abs() <= tol(a.T @ b, a.T.abs() @ b.abs(), 6)).all()


def _long_plan(T):
    from bitsparse_amd.experts import ExpertPlan
    at = torch.arange(T, device="cuda", dtype=torch.int32)
    at[T - 2:] = -1                                                         # two without an expert
    return ExpertPlan(torch.tensor([0, T - 2], device="cuda", dtype=torch.int32), at, at[:, None].clone())


@pytest.mark.parametrize("kept", [False, True])
def test_sums_of_more_tokens_than_a_launch_has(kept):
    """2^24 workgroups of 256 threads are past a launch's 2^32 threads."""
    from bitsparse_amd.experts import expert_combine
    T, D = 2 ** 24 + 3, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    y = torch.randn(T, D, generator=g, device="cuda").to(BF).requires_grad_()
    w = torch.rand(T, 1, generator=g, device="cuda").requires_grad_(kept)
    go = torch.randn(T, D, generator=g, device="cuda").to(BF)
    out = expert_combine(y, w, _long_plan(T))
    want = (y.detach().float() * w.detach()).to(BF)                         # (one product, rounded twice on both sides)
    want[T - 2:] = 0
    right = torch.equal(out, want)
    assert right
    got = torch.autograd.grad(out, [y, w] if kept else [y], go)
    want = (go.float() * w.detach()).to(BF)
    want[T - 2:] = 0
    right = torch.equal(got[0], want)
    assert right
    if kept:
        a, b = go.double(), y.detach().double()
        a[T - 2:] = 0
        assert ((got[1][:, 0].double() - (a * b).sum(1)).abs() <= (D + 1) * 2.0 ** -24 * (a * b).abs().sum(1)).all()


def test_a_block_of_more_rows_than_a_launch_has():
    """Against the same tokens by themselves: products over 8 columns and sums of a row have the same bits in both."""
    from bitsparse_amd.experts import ExpertPlan, ExpertsRelu2
    T, D = 2 ** 24 + 3, 8
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(T, D, generator=g, device="cuda").to(BF)
    w = torch.rand(T, 1, generator=g, device="cuda")
    go = torch.randn(T, D, generator=g, device="cuda").to(BF)
    W1, W2 = (torch.randn(1, D, D, generator=g, device="cuda").to(BF) for _ in range(2))

    def step(at):
        leaves = [t[at].clone().requires_grad_() for t in (x, w)]
        n = leaves[0].shape[0]
        order = torch.arange(n, device="cuda", dtype=torch.int32)
        plan = ExpertPlan(torch.tensor([0, n], device="cuda", dtype=torch.int32), order, order[:, None].clone())
        out = ExpertsRelu2.apply(leaves[0], W1, W2, leaves[1], plan)
        return out.detach(), *torch.autograd.grad(out, leaves, go[at])

    whole = step(slice(None))
    for at in (slice(0, 40), slice(2 ** 22 - 20, 2 ** 22 + 20), slice(2 ** 23 - 20, 2 ** 23 + 20), slice(T - 40, T)):
        for a, b in zip(whole, step(at)):
            assert torch.equal(a[at], b)


def test_routing_of_more_tokens_than_a_launch_has():
    from bitsparse_amd.experts import route
    T = 2 ** 28 + 5
    l = torch.randint(-8, 9, (T, 2), device="cuda", dtype=torch.int8).to(BF).requires_grad_()
    w, ids = route(l, 1, renormalize=False)
    right = torch.equal(ids[:, 0] == 1, l[:, 1] > l[:, 0])
    assert right                                # (nothing that a failure would print element by element)
    gap = (l[:, 0] - l[:, 1]).abs().detach()
    want = 1 / (1 + torch.exp(-gap.float()))
    # (a few roundings of 2^-24 each on both sides)
    assert (w[:, 0].detach() - want).abs().max() < 16 * 2.0 ** -24
    del want, ids
    dl, = torch.autograd.grad(w, l, torch.ones_like(w))
    del w
    for at in (slice(0, 1000), slice(2 ** 27 - 500, 2 ** 27 + 500), slice(T - 1000, T)):
        v = l[at].detach().double()
        s = torch.softmax(v, -1)
        full = s[:, 0] * s[:, 1] * torch.where(v[:, 1] > v[:, 0], -1.0, 1.0)
        want = torch.stack([full, -full], 1)
        # (s to 8 roundings, the difference ds - s to as many of 1)
        assert ((dl[at].double() - want).abs() <= 2.0 ** -8 * want.abs() * 1.02 + 16 * 2.0 ** -24 * s).all()


def test_dropout_past_32_bits():
    from bitsparse_amd.dropout import Dropout, dropout
    T, D = 3, 2 ** 30 + 9
    x = torch.ones(T, D, device="cuda", dtype=BF)
    y = dropout(x, Dropout(0.5, 8, 9))
    small = dropout(x[:, :4096].contiguous(), Dropout(0.5, 8, 9))
    assert torch.equal(y[:, :4096], small)                  # the mask goes by row and column alone
    tail = y[:, -100000:]
    share = (tail == 0).float().mean().item()
    assert abs(share - 0.5) < 0.01 and set(tail.unique().tolist()) == {0.0, 2.0}


@pytest.mark.parametrize("top_k", [1, 2])
def test_a_padded_batch(top_k):
    """Tokens of padding, all of whose logits are -infinity, get zeros, give no gradient and change nobody else's."""
    from bitsparse_amd.dropout import Dropout
    logits, x, W1, W2, go, _ = _parts(T=64)
    logits[50:] = -torch.inf
    x[50:] = torch.nan
    go[50:] = torch.inf
    full = _step(logits, x, W1, W2, go, top_k, Dropout(0.0, 0))
    short = _step(logits[:50], x[:50], W1, W2, go[:50], top_k, Dropout(0.0, 0))
    out, dl, dx, dW1, dW2 = full[0], *full[-4:]
    assert torch.equal(out[:50], short[0]) and (out[50:] == 0).all()
    assert torch.equal(dl[:50], short[-4]) and (dl[50:] == 0).all()
    assert torch.equal(dx[:50], short[-3]) and (dx[50:] == 0).all()
    assert torch.equal(dW1, short[-2]) and torch.equal(dW2, short[-1])
