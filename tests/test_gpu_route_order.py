"""The order in which `route` takes equal experts: -0 and +0 are equal, and of equal values the lower index goes first.

The reference sorts on the CPU, stably, values in which -0 was made +0; where the choice is between the logits, or groups of
them by their one best, the chosen experts have to be the same, without an allowance.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _choice(c, k, groups, top_groups):
    """The k first of c (64 bits, CPU; -infinity: none) among the top_groups groups with the largest best value."""
    c = c + 0.0                         # (-0 + 0 is +0)
    T, E = c.shape
    if top_groups < groups:
        by = c.view(T, groups, -1)
        keep = torch.sort(by.amax(-1), dim=-1, descending=True, stable=True).indices[:, :top_groups]
        kept = torch.zeros(T, groups, dtype=torch.bool).scatter_(1, keep, True)
        c = by.masked_fill(~kept[..., None], -torch.inf).view(T, E)
    top = torch.sort(c, dim=-1, descending=True, stable=True)
    return torch.where(top.values[:, :k] > -torch.inf, top.indices[:, :k], -1).int()


def _route(l, k, **kw):
    from bitsparse_amd.experts import route
    return route(l.cuda(), k, **kw)[1].cpu()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_zeros_of_two_signs(dtype, score):
    for row, k, want in (([-0.0, 0.0], 1, [0]), ([0.0, -0.0], 2, [0, 1]), ([-1.0, -0.0, 0.0, -0.0], 3, [1, 2, 3]),
                         ([-0.0] * 5 + [0.0] * 2, 6, [0, 1, 2, 3, 4, 5]), ([-1.0] * 40 + [-0.0] + [-1.0] * 100 + [0.0], 1, [40])):
        assert _route(torch.tensor([row], dtype=dtype), k, score=score).tolist() == [want], row
    # groups by their one best: both best ones are a zero
    l = torch.full((1, 32), -2.0, dtype=dtype)
    l[0, 13], l[0, 20] = -0.0, 0.0
    assert _route(l, 2, score=score, groups=4, top_groups=1).tolist() == [[13, 8]]


# (experts, choices, groups, groups kept): experts one, four, eight and sixteen to a lane, sixteen and 64 lanes to a token
SIZES = [(2, 1, 1, 1), (16, 3, 1, 1), (60, 6, 1, 1), (64, 6, 8, 3), (128, 8, 8, 3), (160, 4, 8, 2), (256, 8, 8, 4), (256, 64, 1, 1), (300, 5, 1, 1),
         (512, 7, 64, 9), (1024, 33, 16, 5)]


@pytest.mark.parametrize("E,k,groups,top_groups", SIZES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("zeros", [0.01, 0.2, 0.9])
def test_logits_times_a_mask(E, k, groups, top_groups, score, dtype, zeros):
    """Negative logits on a coarse grid times a mask of 0 and 1: the largest are zeros, of either sign, and the rest are ties."""
    g = torch.Generator().manual_seed(E + k)
    l = -(torch.randn(700, E, generator=g) * 4).abs().ceil() / 4
    zero = torch.rand(700, E, generator=g) < zeros
    l = torch.where(zero & (torch.rand(700, E, generator=g) < 0.5), 0.0, l * ~zero)
    at = l == 0
    assert (torch.signbit(l) & at).any() and (~torch.signbit(l) & at).any()
    l = l.to(dtype)
    got = _route(l, k, score=score, groups=groups, top_groups=top_groups)
    assert torch.equal(got, _choice(l.double(), k, groups, top_groups))


@pytest.mark.parametrize("E,k,groups,top_groups", SIZES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_equal_and_close_logits(E, k, groups, top_groups, score, dtype):
    """Logits on a coarse grid, in fp32 some of them a few units of the last place beside, the k-th largest of every second
    token moved to zero: the choice is the logits' own, whichever tokens share a wave."""
    g = torch.Generator().manual_seed(E + k + 1)
    T = 900
    l = (torch.randn(T, E, generator=g) * 4).round() / 4
    if dtype == F32:
        close = torch.rand(T, E, generator=g) < 0.3
        l = torch.where(close, l * (1 + 2.0 ** -22 * torch.randint(-3, 4, (T, E), generator=g)), l)
    l[::2] -= l[::2].topk(k, -1).values[:, -1:]
    l = torch.where((l == 0) & (torch.rand(T, E, generator=g) < 0.5), -0.0, l).to(dtype)
    got = _route(l, k, score=score, groups=groups, top_groups=top_groups)
    assert torch.equal(got, _choice(l.double(), k, groups, top_groups))


@pytest.mark.parametrize("E,k", [(8, 2), (64, 6), (256, 8), (300, 5)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_equal_scores_with_a_bias(E, k, score, dtype):
    """Of equal logits with equal biases the lower index; another choice is right only between sums that are next to each other
    without being equal.  Scores below 1 and biases of up to 2 in magnitude, in 64 bits: the score and its sum with the bias are
    off by a few units of 2^-52 on both sides, a softmax's by up to E of them for its own sum; (E + 8) 2^-52 in all."""
    g = torch.Generator().manual_seed(E)
    T = 1500
    l = ((torch.randn(T, E, generator=g) * 2).round() / 2)
    l = torch.where((l == 0) & (torch.rand(T, E, generator=g) < 0.5), -0.0, l).to(dtype)
    b = (torch.randn(E, generator=g) * 4).round().clamp(-16, 16) / 8
    from bitsparse_amd.experts import route
    ids = route(l.cuda(), k, score=score, bias=b.cuda())[1].cpu()
    # (a value's exponential once, so that equal logits have equal scores)
    values, at = torch.unique(l.double() + 0.0, return_inverse=True)
    e = values.exp()
    s = e[at] / e[at].sum(-1, keepdim=True) if score == "softmax" else (e / (1 + e))[at]
    c = s + b.double()
    want = _choice(c, k, 1, 1)
    gap = (c.gather(1, ids.long()) - c.gather(1, want.long())).abs()
    differ = ids != want
    assert ((gap[differ] > 0) & (gap[differ] < (E + 8) * 2.0 ** -52)).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("renormalize", [False, True])
def test_logits_further_apart_than_their_type_holds(dtype, renormalize):
    """Finite logits whose difference is not: the score is 0, as it is of any that far below the largest."""
    from bitsparse_amd.experts import route
    low = torch.finfo(dtype).min
    l = torch.tensor([[1e38, low, 0.0], [low, 2e38, 1.0], [low, low, low], [0.0, low, 1.0]], dtype=dtype, device="cuda").requires_grad_()
    w, ids = route(l, 3, renormalize=renormalize)
    assert ids.tolist() == [[0, 2, 1], [1, 2, 0], [0, 1, 2], [2, 0, 1]]
    e = torch.tensor(1.0, dtype=torch.float64).exp()
    want = torch.tensor([[1, 0, 0], [1, 0, 0], [1 / 3] * 3, [e / (1 + e), 1 / (1 + e), 0]], dtype=torch.float64)
    # an exponential to two roundings, a sum of three to three, a product and a quotient: eight of 2^-24 at most
    assert ((w.detach().cpu().double() - want).abs() <= 8 * 2.0 ** -24 * want).all()
    dl, = torch.autograd.grad(w, l, torch.tensor([[1.0, 2.0, 3.0]], device="cuda").expand(4, 3).contiguous())
    assert torch.isfinite(dl).all() and (dl[:2] == 0).all() and dl[3, 1] == 0
