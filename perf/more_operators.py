"""MLP blocks as experts -- the routing of tokens, the products of ragged groups
of rows with their experts' weights, the weighted sum back to tokens -- and the
dropout in front of the residual, as cases whose speed is measured.

Four kinds of case:

* ``route``: scores of the experts, the choice for each token, its weights, and
  the order of the chosen (token, choice) pairs by expert;
* ``linear``: rows in that order times their expert's weight matrix;
* ``combine``: the experts' results summed into tokens by the routing weights;
* ``drop``: dropout of a block's output, alone or in the step to the next
  block (residual, gate and the next block's norm).

Each with ``own`` false in plain torch operations in 32 bits, with ``own``
true through the framework's entry points.

Definitions (T tokens, E experts, k choices of each token):

    s       = softmax(logits) or sigmoid(logits);  c = s + bias
    kept    = the `top_groups` groups of consecutive experts whose
              `group_best` largest c have the largest sum
    experts = the k largest c of the kept groups, the largest first
    w       = scale s[experts] / sum(s[experts])  (or scale s[experts])
    order   = the pairs t k + j sorted by expert, equal ones by number; a pair
              whose expert is not in 0..E-1 (padding) has no row
    offsets = first row of each expert;  place[t, j] = row of the pair, or -1
    y[r]    = x[order[r] / k] W[e]^T, or x[r] W[e]^T, for the rows r of expert
              e; 0 in the rows behind the last expert's
    out[t]  = sum over j of w[t, j] y[place[t, j]]

    u[r, i] = half i % 2 of word i / 2 % 4 of Philox 4x32-10 with the seed as
              key and the counter (i / 8, r, offset)
    drop(v) = 0 where u < q, v 65536 / (65536 - q) elsewhere, q = round(65536 p)
    x'      = x + gate drop(y), rounded to the type of x;  h = rms norm of x'

(equal values of c, and of a group's sums: the lowest index first).  Sizes are
those of the repository's benchmark and tests (4096 -> 16384 on 4096 tokens,
256 -> 1024, 768 wide on 8192 tokens) cut into experts, and generic ones.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _route(name, T, E, k, score="softmax", bias=False, groups=1, top_groups=1, best=1, renorm=True, l="fp32", train=True):
    return {"name": name, "kind": "route", "T": T, "E": E, "k": k, "score": score, "bias": bias, "groups": groups,
            "top_groups": top_groups, "best": best, "renorm": renorm, "l": l, "train": train}


def _linear(name, T, E, k, D, N, gather=True, idle=0.0, train=True):
    """`idle`: the share of tokens that are padding and go to no expert."""
    return {"name": name, "kind": "linear", "T": T, "E": E, "k": k, "D": D, "N": N, "gather": gather, "idle": idle,
            "train": train}


def _combine(name, T, E, k, D, idle=0.0, train=True):
    return {"name": name, "kind": "combine", "T": T, "E": E, "k": k, "D": D, "idle": idle, "train": train}


def _drop(name, T, D, p, x="bf16", y="bf16", join=False, train=True):
    return {"name": name, "kind": "drop", "T": T, "D": D, "p": p, "x": x, "y": y, "join": join, "train": train}


def listed():
    return [
        # one token of a model that answers: launch and host latency
        _route("route_one_token", 1, 64, 8, "sigmoid", bias=True, groups=8, top_groups=4, best=2, train=False),
        # two of eight experts for each of a training step's tokens, scores in 16 bits
        _route("route_few_experts", 8192, 8, 2, l="bf16"),
        # many small experts, balanced by a bias, of a few groups only: a long training batch
        _route("route_many_experts", 32768, 256, 8, "sigmoid", bias=True, groups=8, top_groups=4, best=2),
        # the experts of one token: their weights are read once
        _linear("linear_one_token", 1, 64, 8, 4096, 1024, train=False),
        # sizes that end inside every tile, rows no vector load is aligned to, a padded batch, experts with few rows or none
        _linear("linear_odd", 1003, 37, 3, 501, 333, gather=False, idle=0.1),
        # the 768-wide block as eight experts on its 8192 tokens, forward and backward
        _linear("linear_block", 8192, 8, 2, 768, 2048),
        # the 4096 -> 16384 block as experts of an eighth of its width, on a long batch: the product back to 4096
        _linear("linear_large", 16384, 16, 2, 2048, 4096, gather=False),
        # 32 sequences that take one token each
        _combine("combine_decode", 32, 64, 8, 4096, train=False),
        # a training step's tokens
        _combine("combine_large", 16384, 64, 4, 4096),
        # a toy model's block
        _drop("drop_small", 257, 100, 0.1),
        # a long batch: streamed from memory
        _drop("drop_large", 16384, 4096, 0.1),
        # the step between two 768-wide blocks, residual stream in 32 bits
        _drop("drop_join", 8192, 768, 0.2, x="fp32", join=True),
    ]


MAX_ROUTE = 32768 * 256         # T * E
MAX_FLOPS = 16384 * 2 * 2048 * 4096
MAX_WEIGHTS = 16 * 2048 * 4096  # E * D * N
MAX_ROWS = 16384 * 4 * 4096     # T * k * D of a combine
MAX_DROP = 16384 * 4096


def _log(rng, lo, hi):
    """An integer of [lo, hi], its logarithm spread evenly."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A width: any, or a multiple of 64."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.4 else max(lo, v // 64 * 64)


def draw(rng):
    kind = rng.choice(["route", "linear", "linear", "combine", "drop"])
    T = _log(rng, 1, 32768 if kind == "route" else 16384)
    train = T > 256 or rng.random() < 0.5
    if kind == "drop":
        while True:
            D = _size(rng, 16, 8192)
            if T * D <= MAX_DROP:
                break
        x, y = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("fp32", "bf16"), ("fp32", "fp32")])
        join = rng.random() < 0.5
        c = _drop("", T, D, rng.choice([0.05, 0.1, 0.2, 0.5, round(rng.uniform(0.01, 0.9), 3)]), x, y if join else x, join, train)
        del c["name"]
        return c
    while True:
        if kind == "route":
            E = _log(rng, 2, 256)
            k = min(E, _log(rng, 1, 8))
            groups = rng.choice([g for g in (1, 1, 2, 4, 8) if E % g == 0 and E // g >= 2])
            top_groups = rng.randint(1, groups)
            if T * E > MAX_ROUTE or k > top_groups * (E // groups):
                continue
            c = _route("", T, E, k, rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, groups, top_groups,
                       rng.choice([1, 2]), rng.random() < 0.7, rng.choice(["fp32", "fp32", "bf16"]), train)
        else:
            E = _log(rng, 1, 128)
            k = min(E, _log(rng, 1, 8))
            D, N = _size(rng, 16, 8192), _size(rng, 16, 8192)
            idle = rng.choice([0.0, 0.0, 0.15])
            if kind == "combine":
                if T * k * D > MAX_ROWS:
                    continue
                c = _combine("", T, E, k, D, idle, train)
            else:
                if E * D * N > MAX_WEIGHTS or T * k * D * N > MAX_FLOPS:
                    continue
                c = _linear("", T, E, k, D, N, rng.random() < 0.5, idle, train)
        del c["name"]
        return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(g, *shape, mul=1.0, add=0.0):
    return torch.randn(shape, generator=g, device="cuda") * mul + add


def _chosen(case, g):
    """Routed pairs: experts [T, k], different ones for each token, some asked for more than others; -1 for padding,
    which stands at the end."""
    T, E, k = case["T"], case["E"], case["k"]
    experts = (_randn(g, T, E) + 0.3 * _randn(g, E)).topk(k, -1).indices.int()
    experts[T - int(case["idle"] * T):] = -1
    return experts


def _plain_plan(experts, E):
    """offsets [E + 1], order [T k], place [T, k], in plain operations"""
    ids = experts.reshape(-1).long()
    ids = torch.where((ids >= 0) & (ids < E), ids, E)
    by, order = torch.sort(ids, dim=0, stable=True)
    offsets = torch.searchsorted(by, torch.arange(E + 1, device=ids.device)).int()
    row = torch.empty_like(order)
    row[order] = torch.arange(order.numel(), device=ids.device)
    place = torch.where(ids < E, row, -1).int().view(experts.shape)
    return offsets, torch.where(by < E, order, -1).int(), place


def _inputs(case, g):
    kind, st = case["kind"], {}
    if kind == "route":
        T, E = case["T"], case["E"]
        st["logits"] = (_randn(g, T, E) + 0.3 * _randn(g, E)).to(TYPES[case["l"]])
        st["bias"] = _randn(g, E, mul=0.05) if case["bias"] else None
        st["g_w"] = _randn(g, T, case["k"])
    elif kind == "linear":
        T, E, k, D, N = (case[n] for n in ("T", "E", "k", "D", "N"))
        st["plan"] = _plain_plan(_chosen(case, g), E)
        x = _randn(g, T if case["gather"] else T * k, D)
        # tokens after a norm, or a squared ReLU's results
        st["x"] = (x if case["gather"] else x.relu().square()).bfloat16()
        st["W"] = _randn(g, E, N, D, mul=0.02).bfloat16()
        if case["train"]:
            st["g_y"] = _randn(g, T * k, N, mul=0.1).bfloat16()
    elif kind == "combine":
        T, k = case["T"], case["k"]
        experts = _chosen(case, g)
        st["plan"] = _plain_plan(experts, case["E"])
        st["y"] = _randn(g, T * k, case["D"]).bfloat16()
        st["w"] = torch.softmax(_randn(g, T, k), -1)
        if case["train"]:
            st["g_out"] = _randn(g, T, case["D"]).bfloat16()
    else:
        T, D = case["T"], case["D"]
        st["seed"], st["offset"] = (int(v) for v in torch.randint(0, 2 ** 62, (2,), generator=g, device="cuda"))
        st["y"] = _randn(g, T, D).to(TYPES[case["y"]])
        if case["join"]:
            st["x"] = _randn(g, T, D).to(TYPES[case["x"]])
            st["gate"] = _randn(g, D, mul=0.2, add=0.5).to(TYPES[case["x"]])
            st["w_pre"] = _randn(g, D, mul=0.2, add=1.0).to(TYPES[case["x"]])
            st["g_x"] = (_randn(g, T, D) + 0.1 * st["y"].float()).to(TYPES[case["x"]])
            st["g_h"] = _randn(g, T, D).to(TYPES[case["y"]])
        else:
            st["g_y"] = _randn(g, T, D).to(TYPES[case["y"]])
    return st


LEAVES = ("logits", "x", "W", "y", "w", "gate", "w_pre")


def prepare(case, seed):
    st = _inputs(case, torch.Generator(device="cuda").manual_seed(seed))
    st["case"] = case
    st["leaves"] = [n for n in LEAVES if n in st and case["train"]]
    for n in st["leaves"]:
        st[n].requires_grad_()
    if case["kind"] == "linear":
        st["longest"] = int(st["plan"][0].diff().max())
    return st


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _top(c, n):
    """Indices of the n largest along the last dimension, the largest first, equal ones by index"""
    return torch.sort(c, dim=-1, descending=True, stable=True).indices[..., :n]


def _plain_route(st):
    c = st["case"]
    T, E, G = c["T"], c["E"], c["groups"]
    score = (lambda v: torch.softmax(v, -1)) if c["score"] == "softmax" else torch.sigmoid
    # the choice is between values that may lie next to each other
    pick = score(st["logits"].detach().double())
    if c["bias"]:
        pick = pick + st["bias"].double()
    if c["top_groups"] < G:
        by = pick.view(T, G, E // G)
        keep = _top(torch.sort(by, dim=-1, descending=True).values[..., :c["best"]].sum(-1), c["top_groups"])
        mask = torch.zeros(T, G, dtype=torch.bool, device=pick.device).scatter_(1, keep, True)
        pick = by.masked_fill(~mask[..., None], -math.inf).view(T, E)
    experts = _top(pick, c["k"])
    w = score(st["logits"].float()).gather(1, experts)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return w * 2.5, experts.int()


def _plain_linear(st):
    """Rows of each expert in a matrix as long as the longest's, one batched product"""
    c = st["case"]
    offsets, order, _ = st["plan"]
    R, E = order.numel(), c["E"]
    first, count = offsets[:-1].long(), offsets.diff()
    at = torch.arange(st["longest"], device="cuda")
    rows = torch.where(at < count[:, None], first[:, None] + at, R)             # [E, longest]
    x = st["x"].float()
    if c["gather"]:
        x = x[order.long().clamp(min=0) // c["k"]]
    x = torch.cat([x, x.new_zeros(1, c["D"])])
    y = x[rows] @ st["W"].float().mT
    # each row has one place in y, those past the last expert's none
    r = torch.arange(R, device="cuda")
    e = torch.searchsorted(offsets[1:].contiguous().long(), r, right=True)
    real = e < E
    e = e.clamp(max=E - 1)
    i = torch.where(real, r - first[e], 0)
    return torch.where(real[:, None], y[e, i], 0.0).bfloat16()


def _plain_combine(st):
    place = st["plan"][2].long()
    y = st["y"].float()[place.clamp(min=0)]
    return torch.where(place[..., None] >= 0, st["w"][..., None] * y, 0.0).sum(1).bfloat16()


def _mul_hi_lo(a, m):
    """High and low words of a times the constant m, both below 2^32, in 64-bit integers"""
    low = (a & 0xffff) * m
    high = (a >> 16) * m + (low >> 16)
    return high >> 16, (high & 0xffff) << 16 | low & 0xffff


def _philox_round(c, key):
    h0, l0 = _mul_hi_lo(c[0], 0xD2511F53)
    h1, l1 = _mul_hi_lo(c[2], 0xCD9E8D57)
    return h1 ^ c[1] ^ key[0], l1, h0 ^ c[3] ^ key[1], l0


def _plain_kept(T, D, q, seed, offset):
    """Which elements stay, [T, D]"""
    row = torch.arange(T, device="cuda")[:, None]
    col = torch.arange((D + 7) // 8, device="cuda")[None]
    c = (col + 0 * row, row + 0 * col, (offset & 0xffffffff) + 0 * row, (offset >> 32) + 0 * row)
    for i in range(10):
        c = _philox_round(c, ((seed + i * 0x9E3779B9) & 0xffffffff, ((seed >> 32) + i * 0xBB67AE85) & 0xffffffff))
    u = torch.stack([h for v in c for h in ((v & 0xffff).expand(T, -1), (v >> 16).expand(T, -1))], -1)
    return u.reshape(T, -1)[:, :D] >= q


def _plain_drop(st):
    """(x', h) or the dropped values, in 32 bits"""
    c = st["case"]
    q = round(c["p"] * 65536)
    kept = _plain_kept(c["T"], c["D"], q, st["seed"], st["offset"])
    y = torch.where(kept, st["y"].float() * (65536 / (65536 - q)), 0.0)
    if not c["join"]:
        return [y.to(st["y"].dtype)]
    x = st["x"].float() + st["gate"].float() * y
    # h is of x' as stored; the gradient passes the rounding as it is
    x = x + (x.to(st["x"].dtype).float() - x).detach()
    h = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * st["w_pre"].float()
    return [x.to(st["x"].dtype), h.to(st["y"].dtype)]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _results(st):
    """{name: result, the differentiable ones first}, and the gradients that arrive at those"""
    c = st["case"]
    if c["kind"] == "route":
        if own:
            from bitsparse_amd.experts import plan_experts, route
            w, experts = route(st["logits"], c["k"], score=c["score"], bias=st["bias"], groups=c["groups"],
                               top_groups=c["top_groups"], group_best=c["best"], renormalize=c["renorm"], scale=2.5)
            plan = plan_experts(experts, c["E"])
        else:
            w, experts = _plain_route(st)
            plan = _plain_plan(experts, c["E"])
        return {"w": w, "experts": experts, "offsets": plan[0], "order": plan[1], "place": plan[2]}, [st["g_w"]]
    if c["kind"] == "linear":
        if own:
            from bitsparse_amd.experts import ExpertPlan, expert_linear
            return {"y": expert_linear(st["x"], st["W"], ExpertPlan(*st["plan"]), gather=c["gather"])}, [st.get("g_y")]
        return {"y": _plain_linear(st)}, [st.get("g_y")]
    if c["kind"] == "combine":
        if own:
            from bitsparse_amd.experts import ExpertPlan, expert_combine
            return {"out": expert_combine(st["y"], st["w"], ExpertPlan(*st["plan"]))}, [st.get("g_out")]
        return {"out": _plain_combine(st)}, [st.get("g_out")]
    if own:
        from bitsparse_amd.dropout import Dropout, dropout
        drop = Dropout(c["p"], st["seed"], st["offset"])
        if c["join"]:
            from bitsparse_amd.residual import RowNorm, block_join
            out = block_join(st["x"], st["y"], gate=st["gate"], drop=drop, pre=RowNorm(st["w_pre"], None, "rms", EPS))
        else:
            out = [dropout(st["y"], drop)]
    else:
        out = _plain_drop(st)
    if c["join"]:
        return {"x1": out[0], "h": out[1]}, [st["g_x"], st["g_h"]]
    return {"out": out[0]}, [st["g_y"]]


def run(state):
    if not state["case"]["train"]:
        with torch.no_grad():
            return _results(state)[0]
    out, seeds = _results(state)
    grads = torch.autograd.grad(list(out.values())[:len(seeds)], [state[n] for n in state["leaves"]], seeds)
    return {**{n: v.detach() for n, v in out.items()}, **{"d" + n: v for n, v in zip(state["leaves"], grads)}}


def work(case):
    T, train = case["T"], case["train"]
    if case["kind"] == "drop":
        xb, yb = (4 if case[n] == "fp32" else 2 for n in ("x", "y"))
        if not case["join"]:
            return {"bytes": T * case["D"] * 2 * yb * (2 if train else 1), "flops": 0}
        # x, y read, x', h written; backward: x', y and both gradients read, dx and dy written
        return {"bytes": T * case["D"] * (2 * xb + 2 * yb + ((3 * xb + 3 * yb) if train else 0)), "flops": 0}
    E, k = case["E"], case["k"]
    if case["kind"] == "route":
        lb = 4 if case["l"] == "fp32" else 2
        # logits read; weights, experts, order and places written; backward: logits, experts and dw read, dlogits written
        return {"bytes": T * E * lb + T * k * 16 + ((T * E * 2 * lb + T * k * 8) if train else 0), "flops": 0}
    R, D = int(T * (1 - case["idle"])) * k, case["D"]
    if case["kind"] == "combine":
        return {"bytes": (R + T) * D * 2 * (2 if train else 1) + T * k * 8 + (R * D * 2 if train else 0), "flops": 0}
    N = case["N"]
    used = E * (1 - (1 - 1 / E) ** R)        # experts that some row asks for, about
    rows_in = T if case["gather"] else T * k
    data = 2 * (rows_in * D + T * k * N) + 2 * used * D * N
    return {"bytes": int(data + (2 * (2 * rows_in * D + T * k * N) + 2 * (used + E) * D * N if train else 0)),
            "flops": 2 * R * D * N * (3 if train else 1)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, the gradients by their formulas
# ---------------------------------------------------------------------------
def _exact_route(case, st):
    T, E, k, G = (case[n] for n in ("T", "E", "k", "groups"))
    l = st["logits"].double().cpu().numpy()
    if case["score"] == "softmax":
        s = np.exp(l - l.max(-1, keepdims=True))
        s /= s.sum(-1, keepdims=True)
    else:
        s = 1.0 / (1.0 + np.exp(-l))
    c = s + st["bias"].double().cpu().numpy() if case["bias"] else s.copy()
    if case["top_groups"] < G:
        by = c.reshape(T, G, E // G)
        best = np.sort(by, -1)[..., ::-1][..., :case["best"]].sum(-1)
        gone = np.argsort(-best, -1, kind="stable")[:, case["top_groups"]:]
        by[np.arange(T)[:, None], gone] = -np.inf
    experts = np.argsort(-c, -1, kind="stable")[:, :k]
    at = np.arange(T)[:, None]
    chosen = s[at, experts]
    total = chosen.sum(-1, keepdims=True) if case["renorm"] else np.ones((T, 1))
    out = {"w": 2.5 * chosen / total, "experts": experts.astype(np.int32), "offsets": None, "order": None, "place": None}
    if case["train"]:
        g = st["g_w"].double().cpu().numpy()
        if case["renorm"]:
            g = g - (g * chosen).sum(-1, keepdims=True) / total
        ds = np.zeros((T, E))
        ds[at, experts] = 2.5 * g / total
        out["dlogits"] = s * (ds - (ds * s).sum(-1, keepdims=True)) if case["score"] == "softmax" else s * (1 - s) * ds
    return out


def _exact_linear(case, st):
    offsets, order, _ = st["plan"]
    ends, source = offsets.tolist(), (order.long() // case["k"] if case["gather"] else torch.arange(order.numel(), device="cuda"))
    x, W = st["x"].double(), st["W"]
    y = torch.zeros(order.numel(), case["N"], dtype=torch.float64, device="cuda")
    dx, dW = torch.zeros_like(x), torch.zeros(W.shape, dtype=torch.float64, device="cuda")
    for e in range(case["E"]):
        a, b = ends[e], ends[e + 1]
        if a < b:
            xe, We = x[source[a:b]], W[e].double()
            y[a:b] = xe @ We.T
            if case["train"]:
                ge = st["g_y"][a:b].double()
                dx.index_add_(0, source[a:b], ge @ We)
                dW[e] = ge.T @ xe
    return {"y": y, "dx": dx, "dW": dW} if case["train"] else {"y": y}


def _exact_combine(case, st):
    _, order, place = st["plan"]
    n = int((place >= 0).sum())
    token, pair = order[:n].long() // case["k"], order[:n].long()
    w, y = st["w"].double().reshape(-1)[pair], st["y"][:n].double()
    out = {"out": torch.zeros(case["T"], case["D"], dtype=torch.float64, device="cuda").index_add_(0, token, w[:, None] * y)}
    if case["train"]:
        g = st["g_out"].double()[token]
        out["dy"] = torch.zeros(st["y"].shape, dtype=torch.float64, device="cuda")
        out["dy"][:n] = w[:, None] * g
        dw = torch.zeros(case["T"] * case["k"], dtype=torch.float64, device="cuda")
        dw[pair] = (y * g).sum(-1)
        out["dw"] = dw.view(place.shape)
    return out


def _exact_kept(T, D, q, seed, offset):
    c = np.zeros((4, T, (D + 7) // 8), np.uint64)
    c[0], c[1] = np.arange((D + 7) // 8)[None], np.arange(T)[:, None]
    c[2], c[3] = offset % 2 ** 32, offset // 2 ** 32
    key = [seed % 2 ** 32, seed // 2 ** 32]
    low, half = np.uint64(2 ** 32 - 1), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = np.stack([(b >> half) ^ c[1] ^ np.uint64(key[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(key[1]), a & low])
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    words = np.ascontiguousarray(c.astype("<u4").transpose(1, 2, 0))
    return torch.from_numpy(words.view("<u2").reshape(T, -1)[:, :D] >= q).cuda()


def _exact_drop(case, st):
    q = round(case["p"] * 65536)
    m = _exact_kept(case["T"], case["D"], q, st["seed"], st["offset"]).double() * (65536 / (65536 - q))
    y = st["y"].double()
    if not case["join"]:
        out = {"out": m * y}
        if case["train"]:
            out["dy"] = m * st["g_y"].double()
        return out
    gate, w = st["gate"].double(), st["w_pre"].double()
    x1 = (st["x"].double() + gate * m * y).to(st["x"].dtype).double()
    r = 1.0 / ((x1 * x1).mean(-1, keepdim=True) + EPS).sqrt()
    n = x1 * r
    out = {"x1": x1, "h": n * w}
    if case["train"]:
        gh = st["g_h"].double()
        dn = gh * w
        out["dx"] = st["g_x"].double() + r * (dn - n * (dn * n).mean(-1, keepdim=True))
        out["dy"] = out["dx"] * gate * m
        out["dgate"] = (out["dx"] * m * y).sum(0)
        out["dw_pre"] = (gh * n).sum(0)
    return out


def exact(case, seed):
    st = _inputs(case, torch.Generator(device="cuda").manual_seed(seed))
    return {"route": _exact_route, "linear": _exact_linear, "combine": _exact_combine, "drop": _exact_drop}[case["kind"]](case, st)
