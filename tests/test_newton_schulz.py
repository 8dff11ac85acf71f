"""Newton-Schulz orthogonalisation and the Muon step against their definitions
in 64 bits.

Tolerance. The error of a result has the same sources as that of the same
steps in fp32 arithmetic, and grows by the same map. An operand's two fp16
halves carry it to 2^-23, and a product leaves out the two lower halves'
product, 2^-22 at most: together 2^-21 against fp32's 2^-24 an operation. So
the Frobenius norm of the error may be 8 times the one that fp32 arithmetic
shows on the same matrix; where that happens to be small (a single row), a
relative error of 2^-21 a step grows by at most s p'(s) / p(s) < 2.4 near one,
2^-21 (1 + 2.4 + ... + 2.4^4) = 55 * 8 * 2^-24 < 512 * 2^-24. The output's own
rounding adds half a step of every element.
"""
import copy
import math

import pytest
import torch

from learningorchestra_amd.ops import functional as F

U = 2.0 ** -24
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]
CUBIC = (1.5, -0.5, 0.0)


def _exact(g, coeffs, eps):
    x = g.double()
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + eps)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT.contiguous()
    for a, b, c in coeffs:
        s = x @ x.mT.contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if tall else x


def _check(got, g, coeffs=(F.NS_COEFFS,) * 5, eps=1e-7):
    if g.numel() < 2_000_000:   # larger references stay on the GPU
        g = g.cpu()
    flat = [v for t in coeffs for v in t]
    ref = _exact(g, coeffs, eps)
    f32 = F._newton_schulz_ref(g.float(), flat, eps).double()
    norm = torch.linalg.matrix_norm
    half = torch.finfo(g.dtype).eps / 2
    tol = 8 * norm(f32 - ref) + (512 * U + half) * norm(ref) + 1e-12
    if g.dtype == torch.float16:   # steps below the normal range
        tol = tol + 2.0 ** -25 * math.sqrt(ref.shape[-1] * ref.shape[-2])
    err = norm(got.double().to(ref.device) - ref)
    assert bool((err <= tol).all()), f"off by {(err / tol).max():.2f} tolerances"


def _matrix(shape, dtype=torch.float32, device="cpu", seed=0, scale=1e-3):
    gen = torch.Generator().manual_seed(seed)
    m, n = shape[-2:]
    r = max(1, min(m, n) // 4)
    u = torch.randn(*shape[:-1], r, generator=gen)
    v = torch.randn(*shape[:-2], r, n, generator=gen)
    g = u @ v / r + torch.randn(*shape, generator=gen)
    return (g * scale).to(dtype).to(device)


SHAPES = [(1, 1), (1, 5), (7, 1), (2, 3), (8, 8), (16, 40), (63, 65), (64, 64),
          (65, 63), (100, 300), (300, 100), (129, 257), (33, 1000), (512, 24),
          (64, 256), (64, 257), (40, 513), (64, 1024), (1024, 50), (64, 1025),
          (1025, 3)]


@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("device", DEVICES)
def test_orthogonalize(device, dtype, m, n):
    scale = 1.0 if dtype == torch.float16 else 1e-3
    g = _matrix((m, n), dtype, device, scale=scale)
    keep = g.clone()
    o = F.orthogonalize(g)
    assert o.shape == g.shape and o.dtype == dtype and torch.equal(g, keep)
    _check(o, g)


# all tile sizes with whole sums and split ones, what full rounds of the chip
# leave over (2900 x 3000), ragged sides, wide and tall, batches
BIG = [(256, 3136), (512, 3000), (5000, 65), (16, 512, 700), (2900, 3000),
       (40, 300, 1030), (640, 1500), (1500, 640), (1100, 1130), (2050, 2100), (3, 128, 384),
       (2, 4, 90, 70), (64, 130, 260), (70, 257, 129), (256, 96, 30), (300, 20, 700)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", BIG)
def test_large_and_batched(shape):
    g = _matrix(shape, device="cuda")
    o = F.orthogonalize(g)
    _check(o, g)
    assert torch.equal(o, F.orthogonalize(g))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [
    (100, 100, 130), (300, 130, 100), (40, 129, 260), (100, 129, 130),
    (40, 129, 400), (60, 257, 260), (100, 129, 400)])
def test_many_tiles_and_short_sums(shape):
    """More 64 x 64 tiles than run at once, sums of 4 to 16 steps."""
    g = _matrix(shape, torch.bfloat16, "cuda")
    o = F.orthogonalize(g)
    _check(o, g)
    assert torch.equal(o, F.orthogonalize(g))
    assert torch.equal(o[7], F.orthogonalize(g[7:8].expand(shape))[0])


@pytest.mark.parametrize("device", DEVICES)
def test_converges_to_the_nearest_orthogonal_matrix(device):
    """Thirty cubic steps settle: O O^T = 1, and O G^T is positive."""
    g = _matrix((40, 90), device=device, scale=1.0)
    o = F.orthogonalize(g, steps=30, coeffs=CUBIC).double().cpu()
    assert (o @ o.T - torch.eye(40)).abs().max() < 1e-5
    u, _, vh = torch.linalg.svd(g.double().cpu(), full_matrices=False)
    assert (o - u @ vh).abs().max() < 1e-4
    _check(o.float(), g, coeffs=(CUBIC,) * 30)


@pytest.mark.parametrize("device", DEVICES)
def test_coefficients_of_each_step(device):
    g = _matrix((70, 50), device=device)
    coeffs = [(4.0, -6.5, 3.0), (3.5, -5.0, 2.2), CUBIC]
    o = F.orthogonalize(g, steps=3, coeffs=coeffs, eps=1e-8)
    _check(o, g, coeffs=coeffs, eps=1e-8)
    one = F.orthogonalize(g, steps=1, coeffs=[CUBIC])
    _check(one, g, coeffs=[CUBIC])


@pytest.mark.parametrize("device", DEVICES)
def test_more_steps_than_one_block_takes(device):
    g = _matrix((20, 30), device=device)
    _check(F.orthogonalize(g, steps=40, coeffs=CUBIC), g, coeffs=(CUBIC,) * 40)


@pytest.mark.parametrize("device", DEVICES)
def test_rank_and_spread(device):
    """Rank one, and singular values over six decades."""
    gen = torch.Generator().manual_seed(3)
    u = torch.randn(80, 1, generator=gen)
    v = torch.randn(1, 120, generator=gen)
    q1 = torch.linalg.qr(torch.randn(60, 60, generator=gen)).Q
    q2 = torch.linalg.qr(torch.randn(60, 60, generator=gen)).Q
    spread = q1 @ torch.diag(torch.logspace(0, -6, 60)) @ q2
    for g in (u @ v, spread):
        _check(F.orthogonalize(g.to(device)), g)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e18, 1e30])
def test_scales_beyond_fp32_squares(scale):
    """The norm's squares are summed in 64 bits."""
    g = _matrix((50, 60), device="cuda", scale=1.0)
    _check(F.orthogonalize(g * scale, eps=0.0), g, eps=0.0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", [(50, 60), (130, 70)])
@pytest.mark.parametrize("power", [-140, 123])
def test_norms_out_of_range(device, shape, power):
    """Whole numbers times a power of two, the norm (or what divides by it)
    beyond fp32: the scale leaves no trace."""
    gen = torch.Generator().manual_seed(9)
    g = torch.randint(-15, 16, shape, generator=gen).float().to(device)
    far = torch.ldexp(g.double(), torch.tensor(power)).float()
    assert torch.equal(torch.ldexp(far.double(), torch.tensor(-power)).float(), g)
    assert torch.equal(F.orthogonalize(far, eps=0.0),
                       F.orthogonalize(g, eps=0.0))


@pytest.mark.parametrize("device", DEVICES)
def test_outputs_that_overlap_the_input(device):
    buf = _matrix((1, 5 * 6 * 8), device=device).view(-1)
    g = buf[:4 * 48].view(4, 6, 8)
    keep = buf.clone()
    with pytest.raises(ValueError):
        F.orthogonalize(g, out=buf[48:].view(4, 6, 8))
    with pytest.raises(ValueError):
        F.orthogonalize(g[1:], out=buf[8:8 + 3 * 48].view(3, 6, 8))
    assert torch.equal(buf, keep)
    want = F.orthogonalize(g[:2])
    F.orthogonalize(g[:2], out=g[2:])
    assert torch.equal(g[2:], want) and torch.equal(g[:2].reshape(-1), keep[:96])


@pytest.mark.parametrize("device", DEVICES)
def test_sides_end(device):
    for m, n in ((1, 2 ** 20 + 1), (2 ** 20 + 1, 1)):
        with pytest.raises(ValueError):
            F.orthogonalize(torch.zeros(m, n, device=device))
        with pytest.raises(ValueError):
            F.MuonPlan([(0, m, n)], 2 ** 20 + 8, device)


@pytest.mark.parametrize("device", DEVICES)
def test_zero_and_bad_matrices_stay_alone(device):
    g = _matrix((4, 70, 40), device=device)
    want = F.orthogonalize(g)
    g[1] = 0
    g[2, 5, 7] = float("nan")
    o = F.orthogonalize(g)
    assert bool((o[1] == 0).all())
    assert bool(o[2].isnan().all())
    assert torch.equal(o[0], want[0]) and torch.equal(o[3], want[3])
    g[2, 5, 7] = float("inf")
    o = F.orthogonalize(g)
    assert bool(o[2].isnan().all())
    assert torch.equal(o[0], want[0]) and torch.equal(o[3], want[3])


@pytest.mark.parametrize("device", DEVICES)
def test_views_and_outputs(device):
    wide = _matrix((3, 40, 100), device=device)
    g = wide[:, :, 20:77]
    want = F.orthogonalize(g.contiguous())
    assert torch.equal(F.orthogonalize(g), want)
    assert torch.equal(F.orthogonalize(g.mT.contiguous().mT), want)
    assert torch.equal(F.orthogonalize(g[:1].expand(3, 40, 57))[2], want[0])
    out = torch.empty_like(want)
    assert F.orthogonalize(g, out=out) is out and torch.equal(out, want)
    h = g.contiguous()
    F.orthogonalize(h, out=h)
    assert torch.equal(h, want)
    for shape in ((0, 4, 5), (3, 0, 5), (3, 4, 0)):
        e = torch.zeros(shape, device=device)
        assert F.orthogonalize(e).shape == shape


@pytest.mark.parametrize("device", DEVICES)
def test_orthogonalize_refusals(device):
    g = _matrix((6, 9), device=device)
    for call in (
            lambda: F.orthogonalize(g[0]),
            lambda: F.orthogonalize(g.double()),
            lambda: F.orthogonalize(g.long()),
            lambda: F.orthogonalize(g, steps=0),
            lambda: F.orthogonalize(g, steps=2.5),
            lambda: F.orthogonalize(g, eps=-1e-3),
            lambda: F.orthogonalize(g, eps=float("nan")),
            lambda: F.orthogonalize(g, steps=101),
            lambda: F.orthogonalize(g, coeffs=(1.0, 2.0)),
            lambda: F.orthogonalize(g, steps=3, coeffs=[CUBIC] * 2),
            lambda: F.orthogonalize(g, coeffs=(8.0, 8.0, 8.0)),
            lambda: F.orthogonalize(g, coeffs=(float("nan"), 0.0, 0.0)),
            lambda: F.orthogonalize(g, out=torch.empty(9, 6, device=device)),
            lambda: F.orthogonalize(g, out=torch.empty(9, 6, device=device).t()),
            lambda: F.orthogonalize(g, out=torch.empty_like(g).bfloat16())):
        with pytest.raises((ValueError, RuntimeError)):
            call()


@pytest.mark.gpu
def test_workspace_in_groups():
    """A batch whose workspace passes the limit runs in several groups."""
    one = _matrix((2, 1024, 1024), device="cuda")
    g = one[:1].repeat(200, 1, 1)
    g[100] = one[1]
    o = F.orthogonalize(g)
    assert torch.equal(o[0], o[199]) and torch.equal(o[3], o[0])
    _check(o[0], one[0])
    _check(o[100], one[1])


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(64, 512), (128, 640)])
def test_batches_beyond_32_bits(m, n):
    """Tiles, and with them the order of sums, go by the batch's size: equal
    matrices of one batch are equal, those of two batches within tolerance."""
    one = _matrix((2, m, n), torch.bfloat16, "cuda")
    g = one[:1].repeat(2 ** 31 // (m * n) + 2, 1, 1)
    g[-1] = one[1]
    F.orthogonalize(g, out=g)
    assert torch.equal(g[0], g[-2])
    _check(g[0], one[0])
    _check(g[-1], one[1])


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(20, 30), (70, 90)])
def test_arena_beyond_32_bits(m, n):
    """The same step at the arena's start and 2^31 elements on."""
    views, total, st = _arena([(m, n)], "cuda")
    far = {k: torch.empty(2 ** 31 + total, dtype=v.dtype, device="cuda")
           for k, v in st.items()}
    for k in st:
        far[k][2 ** 31:] = st[k]
    F.muon_step(F.MuonPlan(views, total, "cuda"), *st.values(), **KW)
    F.muon_step(F.MuonPlan([(o + 2 ** 31, *r) for o, *r in views],
                           2 ** 31 + total, "cuda"), *far.values(), **KW)
    for k in st:
        assert torch.equal(far[k][2 ** 31:], st[k]), k


@pytest.mark.gpu
def test_more_small_matrices_than_one_launch_takes():
    """A row's direction does not change, and its length follows the
    polynomial: from 1, five steps end at p(p(p(p(p(1)))))."""
    n = (1 << 22) + 5
    g = torch.randn(n, 1, 2, generator=torch.Generator("cuda").manual_seed(1),
                    device="cuda")
    o = F.orthogonalize(g, eps=0.0)
    a, b, c = F.NS_COEFFS
    p = 1.0
    for _ in range(5):
        p = a * p + b * p ** 3 + c * p ** 5
    unit = g.double() / g.double().norm(dim=-1, keepdim=True)
    assert (o.double() - p * unit).abs().max() <= 512 * U * p


@pytest.mark.gpu
def test_other_stream_and_graph():
    g = _matrix((2, 200, 330), device="cuda")
    want = F.orthogonalize(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = F.orthogonalize(g)
    side.synchronize()
    assert torch.equal(o, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = F.orthogonalize(g)
    for seed in range(4):
        g.copy_(_matrix((2, 200, 330), device="cuda", seed=seed))
        want = F.orthogonalize(g)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want)


# ---------------------------------------------------------------- muon step
def _arena(mats, device, gap=16, seed=0):
    """Flat state with gaps (as of biases) before, between and after."""
    views, total = [], gap
    for m, n in mats:
        views.append((total, m, n))
        total += (m * n + 7) // 8 * 8 + gap
    gen = torch.Generator().manual_seed(seed)
    st = {"master": torch.randn(total, generator=gen) * 0.05,
          "grad": torch.randn(total, generator=gen) * 1e-3,
          "mom": torch.randn(total, generator=gen) * 4e-3}
    for off, m, n in views:
        st["grad"][off:off + m * n] = _matrix((m, n), seed=seed + off).view(-1)
    st = {k: v.to(device) for k, v in st.items()}
    st["mirror"] = torch.full((total,), 3.0, dtype=torch.bfloat16,
                              device=device)
    return views, total, st


def _muon_reference(views, st, lr, mu, wd, gscale, nesterov, coeffs, eps):
    """64-bit master and momentum, and their tolerances. Momentum takes three
    fp32 operations. w keeps 4 of them, the step's error is the
    orthogonalisation's, of a U that itself is off by at most 6 u |U| (added
    through the same map as 6 more roundings of X, well inside the 8 times)."""
    d = {k: v.double().cpu() for k, v in st.items()}
    w, mom = d["master"].clone(), d["mom"].clone()
    checks = []
    for off, m, n in views:
        sl = slice(off, off + m * n)
        g = d["grad"][sl] * gscale
        mom[sl] = mu * mom[sl] + g
        u = (g + mu * mom[sl] if nesterov else mom[sl]).view(m, n)
        o = _exact(u, coeffs, eps)
        flat = [v for t in coeffs for v in t]
        f32 = F._newton_schulz_ref(u.float(), flat, eps).double()
        step = lr * math.sqrt(max(1.0, m / n))
        old = w[sl].clone()
        w[sl] = (1 - lr * wd) * old - step * o.reshape(-1)
        tol = step * (8 * (f32 - o).norm() + 512 * U * o.norm()) \
            + 4 * U * (old.norm() + w[sl].norm())
        checks.append((sl, tol))
    return w, mom, checks


MODELS = {
    "one": [(64, 800)],
    "small": [(32, 25), (64, 300), (40, 64), (10, 64), (900, 17)],
    "textcnn": [(128, 384), (128, 512), (128, 640), (8, 384)],
    "mixed": [(1, 1), (3, 50), (200, 31), (64, 64), (65, 129), (1, 77),
              (90, 1)],
}
LARGE = {"wide": [(256, 1152), (512, 2048), (1000, 2048), (2048, 512),
                  (1024, 256), (64, 576)]}
KW = dict(lr=0.02, mu=0.95, wd=0.1, gscale=0.5, nesterov=True, eps=1e-7)


def _muon_check(device, mats, kw):
    views, total, st = _arena(mats, device)
    before = {k: v.clone() for k, v in st.items()}
    plan = F.MuonPlan(views, total, device)
    coeffs = (F.NS_COEFFS,) * 5
    for _ in range(2):   # the second step from the first's state
        w, mom, checks = _muon_reference(views, st, coeffs=coeffs, **kw)
        F.muon_step(plan, st["master"], st["grad"], st["mom"], st["mirror"],
                    **kw)
        inside = torch.zeros(total, dtype=torch.bool)
        for sl, tol in checks:
            inside[sl] = True
            err = (st["master"][sl].double().cpu() - w[sl]).norm()
            assert err <= tol, f"{sl}: off by {err / tol:.2f} tolerances"
        m = st["mom"].double().cpu()
        assert bool(((m - mom).abs()
                     <= 3 * U * (mom.abs() + before["grad"].cpu().abs()
                                 + m.abs()))[inside].all())
        assert torch.equal(st["mirror"].cpu()[inside],
                           st["master"].cpu()[inside].bfloat16())
        for k in before:   # gradients everywhere, and all that lies between
            where = ~inside if k != "grad" else torch.ones_like(inside)
            assert torch.equal(st[k].cpu()[where], before[k].cpu()[where]), k


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", MODELS)
def test_muon_step(device, name):
    _muon_check(device, MODELS[name], KW)


@pytest.mark.gpu
@pytest.mark.parametrize("name", LARGE)
def test_muon_step_large(name):
    _muon_check("cuda", LARGE[name], KW)


@pytest.mark.parametrize("device", DEVICES)
def test_muon_step_plain_momentum(device):
    _muon_check(device, MODELS["mixed"], {**KW, "nesterov": False, "wd": 0.0,
                                          "mu": 0.0, "gscale": 1.0})


@pytest.mark.gpu
def test_muon_step_in_a_graph():
    """Replays continue as the eager steps do, with eager work in between."""
    views, total, a = _arena(MODELS["textcnn"], "cuda")
    b = {k: v.clone() for k, v in a.items()}
    plan = F.MuonPlan(views, total, "cuda")

    def step(st):
        F.muon_step(plan, st["master"], st["grad"], st["mom"], st["mirror"],
                    **KW)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b)
    for seed in range(4):
        new = torch.randn(total, generator=torch.Generator().manual_seed(seed))
        for st in (a, b):
            st["grad"].copy_(new * 1e-3)
        step(a)
        graph.replay()
        torch.cuda.synchronize()
        for k in a:
            assert torch.equal(a[k], b[k]), (seed, k)


@pytest.mark.parametrize("device", DEVICES)
def test_muon_refusals(device):
    for views, total in (([], 64), ([(0, 4, 4), (8, 4, 4)], 64),
                         ([(4, 4, 4)], 64), ([(0, 8, 9)], 64),
                         ([(0, 0, 4)], 64), ([(0, 4)], 64),
                         ([(-8, 4, 4)], 64)):
        with pytest.raises((ValueError, RuntimeError)):
            F.MuonPlan(views, total, device)
    views, total, st = _arena([(8, 8)], device)
    plan = F.MuonPlan(views, total, device)
    args = [st["master"], st["grad"], st["mom"], st["mirror"]]
    for i in range(4):
        bad = list(args)
        bad[i] = bad[i][:-8].clone()
        with pytest.raises(RuntimeError):
            F.muon_step(plan, *bad, lr=0.1)
        if device == "cuda":
            bad[i] = args[i].cpu()
            with pytest.raises(RuntimeError):
                F.muon_step(plan, *bad, lr=0.1)
            bad[i] = args[i].double()
            with pytest.raises(RuntimeError):
                F.muon_step(plan, *bad, lr=0.1)
    with pytest.raises((ValueError, RuntimeError)):
        F.muon_step(plan, *args, lr=0.1, steps=0)
    with pytest.raises((ValueError, RuntimeError)):
        F.muon_step(plan, *args, lr=0.1, eps=-1.0)
    with pytest.raises((ValueError, RuntimeError)):
        F.muon_step(plan, *args, lr=0.1, coeffs=(9.0, 9.0, 9.0))


@pytest.mark.parametrize("device", DEVICES)
def test_copied_plan(device):
    """A copy is a plan of its own that does the same."""
    views, total, a = _arena(MODELS["mixed"], device)
    b = {k: v.clone() for k, v in a.items()}
    plan = F.MuonPlan(views, total, device)
    for st, p in ((a, plan), (b, copy.deepcopy(plan))):
        F.muon_step(p, st["master"], st["grad"], st["mom"], st["mirror"], **KW)
    assert torch.equal(a["master"], b["master"])


@pytest.mark.gpu
def test_two_plans_on_two_streams():
    """Steps of two plans at once, each on its own stream."""
    views, total, a = _arena(MODELS["textcnn"], "cuda")
    states = [a, {k: v.clone() for k, v in a.items()}]
    want = {k: v.clone() for k, v in a.items()}
    plans = [F.MuonPlan(views, total, "cuda") for _ in range(2)]
    one = F.MuonPlan(views, total, "cuda")
    for _ in range(3):
        F.muon_step(one, want["master"], want["grad"], want["mom"],
                    want["mirror"], **KW)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s, p, st in zip(streams, plans, states):
            with torch.cuda.stream(s):
                F.muon_step(p, st["master"], st["grad"], st["mom"],
                            st["mirror"], **KW)
    torch.cuda.synchronize()
    for st in states:
        for k in want:
            assert torch.equal(st[k], want[k]), k


# coefficients of each step; those below the line pass 2^10 or fall below 2^-10
# between steps, so that A's bound is beyond 2^20 or below 2^-20
TAKEN = [[(8e5, 0.0, 0.0)], [(9e-7, 0.0, 0.0)], [(1e-12, 0.0, 0.0)],
         [(0.0, 0.0, 0.0)], [(0.0, 0.0, 0.0), CUBIC],
         [(0.0, 1.0, 0.0), (0.0, 0.0, 1.0)],
         # ---
         [(2000.0, 0.0, 0.0), (0.0005, 0.0, 0.0)],
         [(1e6, 0.0, 0.0), (1e-6, 0.0, 0.0)],
         [(1e-6, 0.0, 0.0), (1e6, 0.0, 0.0)],
         [(1e-5, 0.0, 0.0), (1.5e5, -5e14, 0.0)],
         [(4000.0, -6000.0, 2500.0), (2.5e-4, 0.0, 0.0)]]
REFUSED = [[(1048576.0, 0.0, 0.0)], [(2000.0, 0.0, 0.0), (2000.0, 0.0, 0.0)],
           [(0.0, 1e6, 1e6)], [(1e39, -1e39, 0.0)], [(1e300, 0.0, 0.0)],
           [(float("inf"), 0.0, 0.0)], [(0.0, 0.0, float("nan"))],
           [(9e-7, 0.0, 0.0), (1.0, 0.0, 0.0)], [(9e-13, 0.0, 0.0)],
           [(1e-6, 0.0, 0.0), (2e12, 0.0, 0.0)],
           [(1e-5, 0.0, 0.0), (1.0, 0.0, 1e60)]]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", [(20, 30), (70, 90)])
@pytest.mark.parametrize("coeffs", TAKEN)
def test_coefficients_within_the_limits(device, shape, coeffs):
    g = _matrix(shape, device=device)
    _check(F.orthogonalize(g, steps=len(coeffs), coeffs=coeffs), g, coeffs)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", [(20, 30), (70, 90), (0, 5)])
@pytest.mark.parametrize("coeffs", REFUSED)
def test_coefficients_beyond_the_limits(device, shape, coeffs):
    """The same ones on the CPU and on GPUs."""
    g = torch.zeros(shape, device=device)
    with pytest.raises(ValueError):
        F.orthogonalize(g, steps=len(coeffs), coeffs=coeffs)
    plan = F.MuonPlan([(0, 4, 4)], 16, device)
    st = [torch.ones(16, device=device) for _ in range(3)]
    with pytest.raises(ValueError):
        F.muon_step(plan, *st, st[0].bfloat16(), lr=0.1, steps=len(coeffs),
                    coeffs=coeffs)
    assert all(bool((t == 1).all()) for t in st)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("eps", [0.0, 1e-60])
@pytest.mark.parametrize("shape", [(20, 30), (130, 70)])
def test_zeros_without_an_eps(device, eps, shape):
    """A zero matrix stays zero, and with no gradient a weight only decays,
    also where eps is nothing in fp32. NaN and infinities are no zeros."""
    g = _matrix((3, *shape), device=device)
    want = F.orthogonalize(g, eps=eps)
    g[1] = 0
    o = F.orthogonalize(g, eps=eps)
    assert bool((o[1] == 0).all())
    assert torch.equal(o[0], want[0]) and torch.equal(o[2], want[2])
    for bad in ("nan", "inf"):
        g[1, 2, 3] = float(bad)
        assert bool(F.orthogonalize(g, eps=eps)[1].isnan().all())
    views, total, st = _arena([shape, (5, 9)], device)
    for k in ("grad", "mom"):
        st[k][views[0][0]:views[0][0] + shape[0] * shape[1]] = 0
    old = st["master"].clone()
    F.muon_step(F.MuonPlan(views, total, device), *st.values(),
                **{**KW, "eps": eps})
    sl = slice(views[0][0], views[0][0] + shape[0] * shape[1])
    keep = 1.0 - KW["lr"] * KW["wd"]
    assert (st["master"][sl].double() - keep * old[sl].double()).abs().max() \
        <= 2 * U * old.abs().max()
    assert bool(st["master"].isfinite().all())
