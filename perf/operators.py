"""Workloads of the layer-norm and Muon operators, with their plain forms.

``run`` computes an operator from elementary torch operations where ``own`` is
false, and through ``learningorchestra_amd.ops.functional`` where it is true.

Operators and their definitions (T is the activations' type):

* layer norm over the last axis of x [rows, cols]
      s = x, or round_T(x + residual)
      y = (s - mean) * invstd * gamma + beta,  invstd = (var + eps)^-1/2
  and its backward pass
      xhat = (s - mean) * invstd,  h = dy * gamma
      dx     = invstd * (h - avg(h) - xhat * avg(h * xhat))  (+ dskip)
      dgamma = sum_rows dy * xhat,  dbeta = sum_rows dy
* orthogonalisation of G [batch, m, n] by Newton-Schulz steps
      X = G / (|G|_F + eps);  A = X X^T;  X <- a X + (b A + c A^2) X
* one Muon step of every weight matrix of a flat parameter arena
      mom <- mu mom + g;  U = g + mu mom;  O = orthogonalise(U)
      w <- (1 - lr wd) w - lr max(1, m/n)^1/2 O;  mirror = bf16(w)
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LN_EPS = 1e-5
NS_COEFFS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
NS_EPS = 1e-7
LR, MU, WD = 0.02, 0.95, 0.01

# the text CNN's three convolutions (filters x taps * embedding)
TEXTCNN = "128x384 128x512 128x640"


def _resnet50() -> str:
    # every weight matrix of the ResNet-50 (out channels x taps * in channels,
    # the stem's three input channels padded to 8) with its classifier
    mats = [(64, 49 * 8)]
    cin = 64
    for mid, blocks in ((64, 3), (128, 4), (256, 6), (512, 3)):
        for b in range(blocks):
            mats += [(mid, cin), (mid, 9 * mid), (4 * mid, mid)]
            if b == 0:
                mats.append((4 * mid, cin))
            cin = 4 * mid
    mats.append((1000, 2048))
    return " ".join(f"{m}x{n}" for m, n in mats)


def _ln(name, rows, cols, dtype, residual, train):
    return {"name": name, "op": "layernorm", "rows": rows, "cols": cols,
            "dtype": dtype, "residual": residual, "train": train}


def _ortho(name, batch, m, n, dtype):
    return {"name": name, "op": "orthogonalize", "batch": batch, "m": m,
            "n": n, "dtype": dtype}


def listed():
    return [
        # one text's pooled features (3 x 128 filters) while predicting
        _ln("ln_infer_one_row", 1, 384, "bf16", False, False),
        # a ragged batch of wide fp16 activations joined to a skip path
        _ln("ln_infer_ragged_skip", 1021, 2050, "fp16", True, False),
        # training on fp32 activations with odd sizes on both axes
        _ln("ln_train_odd", 4099, 1001, "fp32", False, True),
        # the text CNN's embeddings at its benchmark's size: 4096 texts of 256
        _ln("ln_train_embeddings", 4096 * 256, 128, "bf16", False, True),
        # a wide residual block's training pass
        _ln("ln_train_wide_skip", 8192, 8192, "bf16", True, True),
        # the MNIST CNN's second convolution: the smallest call of this kind
        _ortho("ortho_mnist_conv", 1, 64, 800, "fp32"),
        # the MNIST CNN's hidden layer, with a bf16 gradient
        _ortho("ortho_mnist_fc", 1, 256, 3136, "bf16"),
        # a tall matrix with odd sides
        _ortho("ortho_tall_odd", 1, 1537, 511, "fp32"),
        # a stack of equal layers at once
        _ortho("ortho_stack", 16, 512, 2048, "fp32"),
        # one large square weight
        _ortho("ortho_large", 1, 4096, 4096, "fp32"),
        # whole-model optimizer steps
        {"name": "muon_textcnn", "op": "muon", "mats": TEXTCNN},
        {"name": "muon_resnet50", "op": "muon", "mats": _resnet50()},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["layernorm", "layernorm", "orthogonalize", "muon"])
    if kind == "layernorm":
        cols = _log_int(rng, 1, 16384)
        rows = _log_int(rng, 1, max(1, min(1 << 20, (1 << 25) // cols)))
        return {"op": "layernorm", "rows": rows, "cols": cols,
                "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "residual": rng.random() < 0.5, "train": rng.random() < 0.6}
    if kind == "orthogonalize":
        m, n = _log_int(rng, 1, 2500), _log_int(rng, 1, 5000)
        if rng.random() < 0.4:
            m, n = n, m
        lo, hi = min(m, n), max(m, n)
        room = 2.0 ** 36 / (3.0 * lo * lo * hi + float(lo) ** 3)
        room = max(1, min(64, int(room)))
        return {"op": "orthogonalize", "batch": _log_int(rng, 1, room),
                "m": m, "n": n, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    mats = []
    for _ in range(rng.randint(1, 24)):
        m, n = _log_int(rng, 2, 1100), _log_int(rng, 2, 2300)
        if rng.random() < 0.3:
            m, n = n, m
        mats.append(f"{m}x{n}")
    return {"op": "muon", "mats": " ".join(mats)}


def _mats(case):
    return [tuple(int(v) for v in t.split("x")) for t in case["mats"].split()]


def _layout(mats):
    # each matrix starts on a multiple of 8 elements, as in the parameter arena
    offs, total = [], 0
    for m, n in mats:
        offs.append(total)
        total += (m * n + 7) // 8 * 8
    return offs, total


def _gradient(gen, batch, m, n):
    # a few strong directions over a floor of noise, as gradients have them
    r = max(1, min(m, n, 8))
    u = torch.randn(batch, m, r, generator=gen, device=DEVICE)
    v = torch.randn(batch, r, n, generator=gen, device=DEVICE)
    noise = torch.randn(batch, m, n, generator=gen, device=DEVICE)
    return (torch.bmm(u, v) * (1.0 / r) + noise) * 1e-3


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    st = {"case": dict(case)}
    if case["op"] == "layernorm":
        rows, cols, t = case["rows"], case["cols"], TYPES[case["dtype"]]
        shift = 0.3 * randn(cols)
        st["x"] = (randn(rows, cols) + shift).to(t)
        st["gamma"] = 1.0 + 0.1 * randn(cols)
        st["beta"] = 0.1 * randn(cols)
        st["residual"] = randn(rows, cols).to(t) if case["residual"] else None
        if case["train"]:
            st["dy"] = randn(rows, cols).to(t)
            st["dskip"] = (randn(rows, cols).to(t) if case["residual"]
                           else None)
        # the buffers that a layer keeps between steps
        x = st["x"]
        st["out"] = torch.empty_like(x)
        st["sum"] = torch.empty_like(x) if case["residual"] else None
        if case["train"]:
            st["mean"] = torch.empty(rows, device=DEVICE)
            st["invstd"] = torch.empty(rows, device=DEVICE)
            st["dx"] = torch.empty_like(x)
            st["dgamma"] = torch.empty(cols, device=DEVICE)
            st["dbeta"] = torch.empty(cols, device=DEVICE)
        return st
    if case["op"] == "orthogonalize":
        g = _gradient(gen, case["batch"], case["m"], case["n"])
        st["g"] = g.to(TYPES[case["dtype"]])
        return st
    mats = _mats(case)
    offs, total = _layout(mats)
    st["master"] = torch.zeros(total, device=DEVICE)
    st["grad"] = torch.zeros(total, device=DEVICE)
    st["mom"] = torch.zeros(total, device=DEVICE)
    for off, (m, n) in zip(offs, mats):
        end = off + m * n
        st["master"][off:end] = randn(m * n) * math.sqrt(2.0 / n)
        st["grad"][off:end] = _gradient(gen, 1, m, n).view(-1)
        st["mom"][off:end] = _gradient(gen, 1, m, n).view(-1) * 4.0
    st["mirror"] = st["master"].to(torch.bfloat16)
    st["views"] = [(off, m, n) for off, (m, n) in zip(offs, mats)]
    if own:
        from learningorchestra_amd.ops import functional as F
        st["plan"] = F.MuonPlan(st["views"], total, DEVICE)
    return st


# ------------------------------------------------------------- plain forms
def _plain_layernorm(st):
    case = st["case"]
    x, gamma, beta = st["x"], st["gamma"], st["beta"]
    s = x
    if st["residual"] is not None:
        s = (x.float() + st["residual"].float()).to(x.dtype)
    sf = s.float()
    mean = sf.mean(1, keepdim=True)
    cent = sf - mean
    invstd = (cent.square().mean(1, keepdim=True) + LN_EPS).rsqrt()
    xhat = cent * invstd
    y = (xhat * gamma + beta).to(x.dtype)
    outs = {"y": y}
    if st["residual"] is not None:
        outs["sum"] = s
    if case["train"]:
        dy = st["dy"].float()
        h = dy * gamma
        d = invstd * (h - h.mean(1, keepdim=True)
                      - xhat * (h * xhat).mean(1, keepdim=True))
        if st["dskip"] is not None:
            d = d + st["dskip"].float()
        outs["dx"] = d.to(x.dtype)
        outs["dgamma"] = (dy * xhat).sum(0)
        outs["dbeta"] = dy.sum(0)
    return outs


def _newton_schulz(x):
    a, b, c = NS_COEFFS
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    x = x.contiguous()
    norm = x.square().sum((-2, -1), keepdim=True).sqrt()
    x = x / (norm + NS_EPS)
    for _ in range(NS_STEPS):
        gram = torch.matmul(x, x.transpose(-2, -1).contiguous())
        poly = b * gram + c * torch.matmul(gram, gram)
        x = a * x + torch.matmul(poly, x)
    return x.transpose(-2, -1) if tall else x


def _plain_muon(st):
    master, mom = st["master"], st["mom"]
    mom.mul_(MU).add_(st["grad"])
    u = st["grad"] + MU * mom
    for off, m, n in st["views"]:
        o = _newton_schulz(u[off:off + m * n].view(m, n))
        w = master[off:off + m * n].view(m, n)
        w.mul_(1.0 - LR * WD).add_(o, alpha=-LR * math.sqrt(max(1.0, m / n)))
    st["mirror"].copy_(master)
    return {"master": master, "mom": mom, "mirror": st["mirror"]}


# ------------------------------------------------------- the framework's own
def _own_layernorm(F, st):
    case = st["case"]
    F.layernorm_fwd(st["x"], st["gamma"], st["beta"], LN_EPS, st["out"],
                    mean=st.get("mean"), invstd=st.get("invstd"),
                    residual=st["residual"], sum_out=st["sum"])
    outs = {"y": st["out"]}
    if st["residual"] is not None:
        outs["sum"] = st["sum"]
    if case["train"]:
        s = st["x"] if st["sum"] is None else st["sum"]
        F.layernorm_bwd(st["dy"], s, st["mean"], st["invstd"], st["gamma"],
                        st["dgamma"], st["dbeta"], st["dx"],
                        dskip=st["dskip"])
        outs["dx"] = st["dx"]
        outs["dgamma"] = st["dgamma"]
        outs["dbeta"] = st["dbeta"]
    return outs


def run(state):
    op = state["case"]["op"]
    if own:
        from learningorchestra_amd.ops import functional as F
        if op == "layernorm":
            return _own_layernorm(F, state)
        if op == "orthogonalize":
            return {"o": F.orthogonalize(state["g"], steps=NS_STEPS,
                                         coeffs=NS_COEFFS, eps=NS_EPS)}
        F.muon_step(state["plan"], state["master"], state["grad"],
                    state["mom"], state["mirror"], lr=LR, mu=MU, wd=WD,
                    steps=NS_STEPS, coeffs=NS_COEFFS, eps=NS_EPS)
        return {"master": state["master"], "mom": state["mom"],
                "mirror": state["mirror"]}
    if op == "layernorm":
        return _plain_layernorm(state)
    if op == "orthogonalize":
        g = state["g"]
        return {"o": _newton_schulz(g.float()).to(g.dtype)}
    return _plain_muon(state)


def _ns_flops(m, n):
    # X X^T and A A^T are symmetric: one triangle each; B X is whole
    lo, hi = min(m, n), max(m, n)
    return NS_STEPS * (3.0 * lo * lo * hi + float(lo) ** 3)


def work(case):
    if case["op"] == "layernorm":
        rows, cols = case["rows"], case["cols"]
        size = 4 if case["dtype"] == "fp32" else 2
        n = rows * cols
        arrays, flops = 2 + (2 if case["residual"] else 0), 8.0
        small = 8 * cols
        if case["train"]:
            # dy in, dx out (and dskip in)
            arrays += 2 + (1 if case["residual"] else 0)
            flops += 14.0
            small += 8 * cols
        return {"bytes": float(arrays * n * size + small), "flops": flops * n}
    if case["op"] == "orthogonalize":
        size = 4 if case["dtype"] == "fp32" else 2
        b, m, n = case["batch"], case["m"], case["n"]
        return {"bytes": float(2 * b * m * n * size),
                "flops": b * _ns_flops(m, n)}
    mats = _mats(case)
    n = sum(m * c for m, c in mats)
    # in: master, grad, momentum; out: master, momentum, mirror
    return {"bytes": float(n * (4 * 5 + 2)),
            "flops": sum(_ns_flops(m, c) for m, c in mats) + 8.0 * n}


# ------------------------------------------------------ definition in 64 bits
def _exact_layernorm(case, st):
    x = st["x"].double()
    outs = {}
    if st["residual"] is not None:
        s = (x + st["residual"].double()).to(st["x"].dtype)
        x = s.double()
    cols = x.shape[1]
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    inv = 1.0 / torch.sqrt(var + LN_EPS)
    z = (x - mean).mul_(inv)
    gam = st["gamma"].double()
    outs["y"] = torch.addcmul(st["beta"].double(), z, gam)
    if st["residual"] is not None:
        outs["sum"] = x
    if case["train"]:
        dy = st["dy"].double()
        p = dy * gam
        c1 = p.sum(1, keepdim=True) / cols
        c2 = torch.linalg.vecdot(p, z).unsqueeze(1) / cols
        dx = p.sub_(c1).addcmul_(z, c2, value=-1.0).mul_(inv)
        if st["dskip"] is not None:
            dx += st["dskip"].double()
        outs["dx"] = dx
        outs["dgamma"] = torch.linalg.vecdot(dy, z, dim=0)
        outs["dbeta"] = dy.sum(0)
    return outs


def _exact_orthogonal(g):
    # (a + b S + c S^2) X with S = X X^T, or X (a + b S + c S^2) with
    # S = X^T X, whichever is the smaller
    a, b, c = NS_COEFFS
    x = g / (torch.linalg.matrix_norm(g)[..., None, None] + NS_EPS)
    left = x.shape[-2] <= x.shape[-1]
    eye = torch.eye(min(x.shape[-2:]), dtype=torch.float64, device=x.device)
    for _ in range(NS_STEPS):
        xt = x.mT.contiguous()
        s = x @ xt if left else xt @ x
        q = a * eye + s @ (b * eye + c * s)
        x = q @ x if left else x @ q
    return x


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "layernorm":
        return _exact_layernorm(case, st)
    if case["op"] == "orthogonalize":
        return {"o": _exact_orthogonal(st["g"].double())}
    g = st["grad"].double()
    mom = st["mom"].double() * MU + g
    u = g + MU * mom
    w = st["master"].double() * (1.0 - LR * WD)
    for off, m, n in st["views"]:
        end = off + m * n
        o = _exact_orthogonal(u[off:end].reshape(m, n))
        w[off:end] -= LR * math.sqrt(max(1.0, m / n)) * o.reshape(-1)
    return {"master": w, "mom": mom, "mirror": w}
