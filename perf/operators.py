"""The operators around the MLP block -- the norms before and after it with its
gate and residual scale, and the orthogonalised update of its weight
matrices -- as cases whose speed is measured.

Four kinds of case:

* ``norm``: the norm in front of a block, h = norm(x);
* ``join``: the step from one block to the next, x' = scale x + gate norm(y)
  and h = norm(x') for the next block;
* ``ortho``: the orthogonal factor of a gradient by Newton-Schulz products;
* ``muon``: the whole update of a set of weight matrices: momentum,
  orthogonalisation, weight decay and step.

Each with ``own`` false in plain torch operations in 32 bits, with ``own``
true through the framework's entry points.

Definitions (sums over a row's D elements; c(v) = v - mean(v) for a layer
norm, v for an RMS norm):

    norm(v) = c(v) / sqrt(mean(c(v)^2) + eps) * weight + bias
    x'      = scale * x + gate * norm(y), rounded to the type of x
    h       = norm(x') of x' as it is stored, in the type of y
    M'      = mu M + (1 - mu) G;  U = (1 - mu) G + mu M' (Nesterov)
    X_0     = U / (||U||_F + eps)
    X_k+1   = a X_k + (b A + c A^2) X_k,  A = X_k X_k^T  (of the transpose
              where there are more rows than columns)
    W'      = (1 - lr decay) W - lr s X_5,  s = 0.2 sqrt(max(rows, columns))

Sizes are those of the repository's benchmark, tests and configurations (the
768 -> 3072 block on 8192 tokens and its stack of 12, the 4096 -> 16384 block
on 4096 tokens, the tests' 256 -> 1024 block) and generic ones around them.
"""
import math

import torch

own = False

STEPS = 5
COEF = (3.4445, -4.7750, 2.0315)
NS_EPS = 1e-7
NORM_EPS = 1e-5
MU, LR, DECAY = 0.95, 3e-4, 0.1

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _norm(name, T, D, norm, x="bf16", h="bf16", bias=False, train=True):
    return {"name": name, "kind": "norm", "T": T, "D": D, "norm": norm, "x": x, "h": h, "bias": bias, "train": train}


def _join(name, T, D, norm, x="bf16", h="bf16", bias=False, gate="channel", scale="channel", train=True):
    return {"name": name, "kind": "join", "T": T, "D": D, "norm": norm, "x": x, "h": h, "bias": bias, "gate": gate,
            "scale": scale, "train": train}


def _ortho(name, B, R, C, g="bf16", like="grad"):
    return {"name": name, "kind": "ortho", "B": B, "R": R, "C": C, "g": g, "like": like}


def _muon(name, pairs, D, H, g="bf16", w="bf16", m="fp32"):
    """`pairs` MLP blocks: W1 [H, D] and W2 [D, H] of each."""
    return {"name": name, "kind": "muon", "pairs": pairs, "D": D, "H": H, "g": g, "w": w, "m": m}


def listed():
    return [
        # the first norm of a model that answers with one token at a time: launch and host latency
        _norm("norm_one_token", 1, 4096, "rms", train=False),
        # the layer norm in front of the 768-wide block on its 8192 tokens, forward and backward
        _norm("norm_block_layer", 8192, 768, "layer", bias=True),
        # between two blocks when 32 sequences each take one token
        _join("join_decode", 32, 4096, "rms", train=False),
        # between two 768-wide blocks in training
        _join("join_block", 8192, 768, "rms"),
        # a residual stream in 32 bits, layer norms with biases, a gate for each token, a learned scalar for
        # the residual, rows that no vector load is aligned to
        _join("join_odd_fp32", 3005, 2501, "layer", x="fp32", bias=True, gate="token", scale="scalar"),
        # a long batch of a 4096-wide model: streamed from memory
        _join("join_large", 16384, 4096, "rms"),
        # the gradient of a test-sized block's weight: launches only
        _ortho("ortho_small", 1, 256, 1024),
        # sizes that end inside every tile, more rows than columns, a 32-bit gradient
        _ortho("ortho_odd_tall", 1, 2731, 1001, g="fp32"),
        # one weight of the 4096 -> 16384 block
        _ortho("ortho_large", 1, 4096, 16384),
        # a toy model's optimiser step
        _muon("muon_small", 2, 256, 1024),
        # the optimiser step of the stack of 12 blocks of 768 -> 3072
        _muon("muon_stack", 12, 768, 3072),
        # weights and gradients in 32 bits, square-ish, momentum in 16
        _muon("muon_fp32", 1, 2048, 5500, g="fp32", w="fp32", m="bf16"),
    ]


MAX_ROWS = 16384 * 4096                         # T * D of a drawn norm or join
MAX_FLOPS = 3 * 4096 ** 2 * 16384 + 4096 ** 3   # of one Newton-Schulz step of a drawn ortho or muon


def _log(rng, lo, hi):
    """An integer of [lo, hi], its logarithm spread evenly."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A width: any, or a multiple of 64."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.4 else max(lo, v // 64 * 64)


def draw(rng):
    kind = rng.choice(["norm", "join", "join", "ortho", "muon"])
    if kind in ("norm", "join"):
        while True:
            T, D = _log(rng, 1, 16384), _size(rng, 64, 8192)
            if T * D <= MAX_ROWS:
                break
        x, h = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("fp32", "bf16"), ("fp32", "fp32")])
        norm, bias = rng.choice(["rms", "layer"]), rng.random() < 0.5
        train = T > 256 or rng.random() < 0.5
        if kind == "norm":
            c = _norm("", T, D, norm, x, h, bias, train)
        else:
            c = _join("", T, D, norm, x, h, bias, rng.choice(["channel", "channel", "token", "scalar", "full"]),
                      rng.choice(["channel", "scalar"]), train)
    else:
        while True:
            a, b = _size(rng, 32, 4096), _size(rng, 32, 16384)
            B = _log(rng, 1, 24)
            n = B * _step_flops(a, b) * (2 if kind == "muon" else 1)
            if n <= MAX_FLOPS and max(a, b) <= 64 * min(a, b):
                break
        if kind == "ortho":
            c = _ortho("", B, a, b, rng.choice(["bf16", "fp32"]), rng.choice(["grad", "normal"]))
        else:
            c = _muon("", B, a, b, rng.choice(["bf16", "fp32"]), rng.choice(["bf16", "fp32"]),
                      rng.choice(["bf16", "fp32"]))
    del c["name"]
    return c


def _step_flops(a, b):
    """One Newton-Schulz step: two symmetric products at half their operations and one whole."""
    m, n = min(a, b), max(a, b)
    return 3 * m * m * n + m ** 3


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(g, *shape, mul=1.0, add=0.0):
    return torch.randn(shape, generator=g, device="cuda") * mul + add


def _rows_inputs(case, g):
    """A residual stream whose channels have scales and offsets of their own, a block's output, learned vectors
    near their initial values, and the gradients of both results."""
    T, D = case["T"], case["D"]
    xt, ht = TYPES[case["x"]], TYPES[case["h"]]
    vec = lambda mul, add: _randn(g, D, mul=mul, add=add).to(xt)  # noqa: E731
    st = {"x": (_randn(g, T, D) * torch.exp(0.5 * _randn(g, D)) + 0.3 * _randn(g, D)).to(xt)}
    st["w_pre"] = vec(0.2, 1.0)
    st["b_pre"] = vec(0.1, 0.0) if case["bias"] else None
    if case["kind"] == "join":
        st["y"] = (_randn(g, T, D, mul=0.7) + 0.2 * _randn(g, D)).to(ht)
        st["w_post"] = vec(0.2, 1.0)
        st["b_post"] = vec(0.1, 0.0) if case["bias"] else None
        shape = {"channel": (D,), "token": (T, 1), "scalar": (1,), "full": (T, D)}[case["gate"]]
        st["gate"] = _randn(g, *shape, mul=0.2, add=0.5).to(ht if case["gate"] == "full" else xt)
        st["scale"] = _randn(g, D if case["scale"] == "channel" else 1, mul=0.05, add=0.95).to(xt)
        # what a gradient has in common with the values it belongs to keeps its sums over all of them away from 0
        st["g_x"] = (_randn(g, T, D) + 0.1 * st["x"].float() + 0.1 * st["y"].float()).to(xt)
    st["g_h"] = _randn(g, T, D).to(ht)
    return st


def _matrices(g, B, R, C, like):
    """Weight gradients: of a Linear whose inputs are a ReLU's with channels of their own rate and whose outputs'
    gradients have channels of their own scale, summed over tokens; or independent normal values."""
    if like == "normal":
        return _randn(g, B, R, C, mul=1e-3)
    T = 2 * min(R, C) + 64
    dy = _randn(g, B, T, R) * torch.exp(0.5 * _randn(g, B, 1, R))
    r = torch.relu(_randn(g, B, T, C) + 0.3 * _randn(g, B, 1, C))
    return torch.bmm(dy.mT.contiguous(), r) * (1e-3 / math.sqrt(T))


def _muon_inputs(case, g):
    """Weights, gradients and momenta, each as W1 of every block [pairs, H, D] and W2 of every block [pairs, D, H]"""
    st = {"W": [], "G": [], "M": []}
    for R, C in ((case["H"], case["D"]), (case["D"], case["H"])):
        n = case["pairs"]
        st["W"].append(_randn(g, n, R, C, mul=0.02).to(TYPES[case["w"]]))
        st["G"].append(_matrices(g, n, R, C, "grad").to(TYPES[case["g"]]))
        st["M"].append((0.5 * _matrices(g, n, R, C, "grad")).to(TYPES[case["m"]]))
    return st


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = {"case": case}
    if case["kind"] in ("norm", "join"):
        st.update(_rows_inputs(case, g))
        if case["train"]:
            st["leaves"] = [k for k in ("x", "y", "w_pre", "b_pre", "w_post", "b_post", "gate", "scale")
                            if st.get(k) is not None]
            for k in st["leaves"]:
                st[k].requires_grad_()
    elif case["kind"] == "ortho":
        G = _matrices(g, case["B"], case["R"], case["C"], case["like"]).to(TYPES[case["g"]])
        st["G"] = G if case["B"] > 1 else G[0]
    else:
        st.update(_muon_inputs(case, g))
        # the lists of parameters, gradients and buffers that an optimiser goes through
        st["lists"] = [[t for stack in st[k] for t in stack.unbind(0)] for k in ("W", "G", "M")]
    return st


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_norm(v, kind, weight, bias):
    """norm of the rows of v, in 32 bits"""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    n = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + NORM_EPS) * weight.float()
    return n if bias is None else n + bias.float()


def _plain_rows(st):
    """(x', h) in 32 bits; x' None for a norm alone"""
    c = st["case"]
    x, x1 = st["x"].float(), None
    if c["kind"] == "join":
        p = _plain_norm(st["y"].float(), c["norm"], st["w_post"], st["b_post"])
        x = st["scale"].float() * x + st["gate"].float() * p
        # h is of x' as stored; the gradient passes the rounding as it is
        x1 = x = x + (x.to(st["x"].dtype).float() - x).detach()
    return x1, _plain_norm(x, c["norm"], st["w_pre"], st["b_pre"])


def _plain_orthogonal(U):
    """The orthogonal factor of each matrix of U [B, R, C], in 32 bits"""
    tall = U.shape[-2] > U.shape[-1]
    X = U.mT.contiguous() if tall else U
    X = X / (X.square().sum((-2, -1), keepdim=True).sqrt() + NS_EPS)
    a, b, c = COEF
    for _ in range(STEPS):
        A = X @ X.mT
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.mT if tall else X


def _plain_muon(W, G, M):
    """W and M, stacks of equally shaped matrices, updated in place"""
    G = G.float()
    M.copy_(MU * M.float() + (1 - MU) * G)
    X = _plain_orthogonal((1 - MU) * G + MU * M.float())
    s = 0.2 * math.sqrt(max(X.shape[-2:]))
    W.copy_((1 - LR * DECAY) * W.float() - LR * s * X)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _run_rows(st):
    c = st["case"]
    if own:
        from bitsparse_amd.residual import RowNorm, block_join, block_norm
        pre = RowNorm(st["w_pre"], st["b_pre"], c["norm"], NORM_EPS)
        if c["kind"] == "norm":
            x1, h = None, block_norm(st["x"], pre, dtype=TYPES[c["h"]])
        else:
            post = RowNorm(st["w_post"], st["b_post"], c["norm"], NORM_EPS)
            x1, h = block_join(st["x"], st["y"], post=post, gate=st["gate"], scale=st["scale"], pre=pre)
    else:
        x1, h = _plain_rows(st)
        h = h.to(TYPES[c["h"]])
        x1 = None if x1 is None else x1.to(TYPES[c["x"]])
    out = {"h": h.detach()}
    if x1 is not None:
        out["x1"] = x1.detach()
    if c["train"]:
        ends, seeds = ([h], [st["g_h"]]) if x1 is None else ([x1, h], [st["g_x"], st["g_h"]])
        grads = torch.autograd.grad(ends, [st[k] for k in st["leaves"]], seeds)
        out.update({"d" + k: v for k, v in zip(st["leaves"], grads)})
    return out


def run(state):
    kind = state["case"]["kind"]
    if kind in ("norm", "join"):
        if state["case"]["train"]:
            return _run_rows(state)
        with torch.no_grad():
            return _run_rows(state)
    if kind == "ortho":
        G = state["G"]
        if own:
            from bitsparse_amd.muon import orthogonalize
            return {"O": orthogonalize(G, steps=STEPS, coefficients=COEF, eps=NS_EPS)}
        return {"O": _plain_orthogonal(G.float().reshape(-1, *G.shape[-2:])).reshape(G.shape).to(torch.bfloat16)}
    if own:
        from bitsparse_amd.muon import muon_update_
        muon_update_(*state["lists"], lr=LR, momentum=MU, nesterov=True, weight_decay=DECAY, adjust="rms", steps=STEPS,
                     coefficients=COEF, eps=NS_EPS)
    else:
        _plain_muon(state["W"][0], state["G"][0], state["M"][0])
        _plain_muon(state["W"][1], state["G"][1], state["M"][1])
    return {"W": state["W"], "M": state["M"]}


def work(case):
    if case["kind"] in ("norm", "join"):
        n = case["T"] * case["D"]
        xb, hb = (4 if case[k] == "fp32" else 2 for k in ("x", "h"))
        gate = hb if case.get("gate") == "full" else 0
        join = case["kind"] == "join"
        # forward: x (y, gate) read, (x') and h written
        total = n * (xb + hb + ((xb + hb + gate) if join else 0))
        if case["train"]:
            # backward: x or x' and the gradient of h read, dx written; a join: x (the scale's gradient), y, the
            # gradient of x' and the gate read, dy and the gate's gradient written
            total += n * (2 * xb + hb + ((2 * xb + 2 * hb + 2 * gate) if join else 0))
        return {"bytes": total, "flops": 0}
    if case["kind"] == "ortho":
        n = case["B"] * case["R"] * case["C"]
        return {"bytes": n * ((4 if case["g"] == "fp32" else 2) + 2),
                "flops": STEPS * case["B"] * _step_flops(case["R"], case["C"])}
    n = 2 * case["pairs"] * case["D"] * case["H"]
    size = {k: 4 if case[k] == "fp32" else 2 for k in ("g", "w", "m")}
    return {"bytes": n * (size["g"] + 2 * size["w"] + 2 * size["m"]),
            "flops": STEPS * 2 * case["pairs"] * _step_flops(case["D"], case["H"])}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, the gradients by their formulas
# ---------------------------------------------------------------------------
def _standard(v, layer):
    """(v centred and divided by its deviation, 1 / deviation) by rows"""
    c = v - v.mean(-1, keepdim=True) if layer else v
    r = 1.0 / ((c * c).mean(-1, keepdim=True) + NORM_EPS).sqrt()
    return c * r, r


def _standard_grad(dn, n, r, layer):
    """The gradient of v from that of its standard form n"""
    d = dn - n * (dn * n).mean(-1, keepdim=True)
    return r * (d - dn.mean(-1, keepdim=True) if layer else d)


def _d(t):
    return None if t is None else t.detach().double()


def _exact_rows(case, st):
    layer, join = case["norm"] == "layer", case["kind"] == "join"
    v = {k: _d(st.get(k)) for k in ("x", "y", "w_pre", "b_pre", "w_post", "b_post", "gate", "scale", "g_x", "g_h")}
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    out, x1 = {}, v["x"]
    if join:
        yn, yr = _standard(v["y"], layer)
        p = yn * v["w_post"] + (zero if v["b_post"] is None else v["b_post"])
        x1 = (v["scale"] * v["x"] + v["gate"] * p).to(st["x"].dtype).double()
        out["x1"] = x1
    xn, xr = _standard(x1, layer)
    out["h"] = xn * v["w_pre"] + (zero if v["b_pre"] is None else v["b_pre"])
    if not case["train"]:
        return out
    out["dw_pre"] = (v["g_h"] * xn).sum(0)
    if case["bias"]:
        out["db_pre"] = v["g_h"].sum(0)
    total = _standard_grad(v["g_h"] * v["w_pre"], xn, xr, layer)
    if not join:
        out["dx"] = total
        return out
    total = total + v["g_x"]
    out["dx"] = total * v["scale"]
    out["dscale"] = (total * v["x"]).sum(0) if case["scale"] == "channel" else (total * v["x"]).sum().reshape(1)
    dg = total * p
    out["dgate"] = {"channel": lambda: dg.sum(0), "token": lambda: dg.sum(1, keepdim=True),
                    "scalar": lambda: dg.sum().reshape(1), "full": lambda: dg}[case["gate"]]()
    dp = total * v["gate"]
    out["dw_post"] = (dp * yn).sum(0)
    if case["bias"]:
        out["db_post"] = dp.sum(0)
    out["dy"] = _standard_grad(dp * v["w_post"], yn, yr, layer)
    return out


def _exact_orthogonal(U):
    """The Newton-Schulz factor of one matrix, step by step"""
    wide = U.shape[0] <= U.shape[1]
    X = U if wide else U.T
    X = X / (torch.linalg.matrix_norm(X) + NS_EPS)
    a, b, c = COEF
    eye = torch.eye(X.shape[0], dtype=torch.float64, device="cuda")
    for _ in range(STEPS):
        A = X @ X.T
        X = (a * eye + A @ (b * eye + c * A)) @ X
    return X if wide else X.T


def exact(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] in ("norm", "join"):
        return _exact_rows(case, _rows_inputs(case, g))
    if case["kind"] == "ortho":
        G = _matrices(g, case["B"], case["R"], case["C"], case["like"]).to(TYPES[case["g"]]).double()
        O = torch.stack([_exact_orthogonal(G[i]) for i in range(case["B"])])
        return {"O": O if case["B"] > 1 else O[0]}
    st, out = _muon_inputs(case, g), {"W": [], "M": []}
    for W, G, M in zip(st["W"], st["G"], st["M"]):
        W, G = W.double(), G.double()
        new = MU * M.double() + (1 - MU) * G
        new = new.to(M.dtype).double() if case["m"] == "bf16" else new
        O = torch.stack([_exact_orthogonal(u) for u in (1 - MU) * G + MU * new])
        out["M"].append(new)
        out["W"].append((1 - LR * DECAY) * W - LR * 0.2 * math.sqrt(max(W.shape[-2:])) * O)
    return out
