"""Newton-Schulz steps against their definition in 64 bits, with tolerances
that take nothing from the code under test, row by row, and with split sums.

The yardstick is `_steps32`: the same steps in fp32, written from the
definition. Its own distance from 64 bits is bounded too: each of a step's
three products sums K values, off by sqrt(K) u in the norm if roundings fall
at random (u = 2^-24), and the map s -> a s + b s^3 + c s^5 grows that by
max |p'| over the singular values in each later step. The quintic's are at most
1.21 after a step, where |p'| < 3.96, and 1 + 3.96 + ... + 3.96^4 < 330; norms
fall by less than 1.8 on the way to the end. So 3 * 330 * 1.8 < 1800 times
sqrt(K) u.

A result may be off by 8 times the yardstick (two fp16 halves keep an operand
to 2^-23 and leave out 2^-22 of a product: 2^-21 against fp32's 2^-24), by
512 u where the yardstick is small by chance (55 * 8 u: 2^-21 a step, grown by
s p'(s) / p(s) < 2.4 a step near one), and by the output's own rounding.
"""
import math
import os
import subprocess

import pytest
import torch

from learningorchestra_amd.ops import functional as F

U = 2.0 ** -24
QUINTIC = (3.4445, -4.7750, 2.0315)
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _steps(g, dtype, steps=5, eps=1e-7):
    """The definition: X = G / (|G| + eps), X <- a X + b A X + c A (A X)."""
    x = g.double()
    x = (x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)).to(dtype)
    tall = x.shape[-2] > x.shape[-1]
    x = (x.mT if tall else x).contiguous()
    a, b, c = QUINTIC
    for _ in range(steps):
        gram = torch.matmul(x, x.mT.contiguous())
        ax = torch.matmul(gram, x)
        x = a * x + b * ax + c * torch.matmul(gram, ax)
    return x.mT if tall else x


def _check(got, g):
    g = g.cpu() if g.numel() < 2_000_000 else g
    ref = _steps(g, torch.float64)
    norm = torch.linalg.matrix_norm
    yard = norm(_steps(g, torch.float32).double() - ref)
    size = norm(ref)
    assert bool((yard <= 1800 * math.sqrt(max(g.shape[-2:])) * U * size).all())
    tol = 8 * yard + (512 * U + torch.finfo(got.dtype).eps / 2) * size + 1e-12
    if got.dtype == torch.float16:   # steps below the normal range
        tol = tol + 2.0 ** -25 * math.sqrt(g.shape[-1] * g.shape[-2])
    err = norm(got.double().to(ref.device) - ref)
    assert bool((err <= tol).all()), f"off by {(err / tol).max():.2f} tolerances"


def _matrix(shape, dtype=torch.float32, device="cpu", seed=0):
    gen = torch.Generator().manual_seed(seed)
    m, n = shape[-2:]
    r = max(1, min(m, n) // 4)
    u = torch.randn(*shape[:-1], r, generator=gen)
    v = torch.randn(*shape[:-2], r, n, generator=gen)
    g = u @ v / r + torch.randn(*shape, generator=gen)
    return g.to(dtype).to(device)


SHAPES = [(1, 7), (9, 2), (16, 16), (64, 65), (65, 64), (33, 500), (300, 100),
          (64, 1024), (129, 640), (1000, 70), (3, 40, 90), (2, 130, 200)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("device", DEVICES)
def test_orthogonalize(device, dtype, shape):
    g = _matrix(shape, dtype, device)
    _check(F.orthogonalize(g), g)


@pytest.mark.parametrize("mistake", ["c", "b", "a", "norm", "steps"])
def test_the_tolerance_tells_mistakes(mistake):
    """A definition that is a tenth of a per cent off in one place fails."""
    g = _matrix((60, 90))
    a, b, c = QUINTIC
    wrong = {"a": (a * 1.001, b, c), "b": (a, b * 1.001, c),
             "c": (a, b, c * 1.001)}.get(mistake, QUINTIC)
    x = g.double()
    x = x / (x.norm() * (1.001 if mistake == "norm" else 1.0) + 1e-7)
    for _ in range(4 if mistake == "steps" else 5):
        s = x @ x.T
        x = wrong[0] * x + (wrong[1] * s + wrong[2] * (s @ s)) @ x
    with pytest.raises(AssertionError):
        _check(x.float(), g)


# batches whose X X^T is split among blocks, without a table of tasks: its
# tiles' size and in how many parts its sums are, by the plan
SPLIT = {(2, 70, 1100): (32, 3), (5, 9000, 65): (32, 5),
         (2, 256, 3136): (32, 3), (4, 4000, 128): (32, 6),
         (3, 300, 4000): (64, 4), (2, 900, 9000): (64, 5),
         (3, 1200, 4000): (128, 3), (4, 9000, 900): (128, 5)}


def test_batches_that_are_split(tmp_path):
    """The plan's host code, compiled by itself."""
    csrc = os.path.join(os.path.dirname(F.__file__), "..", "csrc")
    rocm = os.environ.get("ROCM_HOME") or os.environ.get("ROCM_PATH") \
        or "/opt/rocm"
    src = tmp_path / "plan.cpp"
    src.write_text("""
#include <cstdio>
#include <cstdlib>
#include "newton_schulz_plan.h"
int main(int n, char** v) {
  for (int i = 1; i + 2 < n; i += 3) {
    const auto mats = lo::ns_plan({{atol(v[i + 1]), atol(v[i + 2])}}, atol(v[i]));
    std::printf("%d %d ", mats[0].kind[lo::NS_GRAM].tile,
                mats[0].kind[lo::NS_GRAM].splits);
  }
}
""")
    exe = str(tmp_path / "plan")
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__",
                    "-I", csrc, "-I", os.path.join(rocm, "include"), str(src),
                    "-o", exe], check=True, capture_output=True)
    args = [str(v) for shape in SPLIT for v in shape]
    out = subprocess.run([exe, *args], check=True, capture_output=True).stdout
    got = [int(v) for v in out.split()]
    assert got == [v for shares in SPLIT.values() for v in shares]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SPLIT)
def test_split_batches(shape):
    """Matrices of their own, so that parts of one in another's place show; the
    last one alone, and twice the same bits."""
    g = _matrix(shape, device="cuda")
    g *= torch.logspace(-2, 2, shape[0], device="cuda").view(-1, 1, 1)
    o = F.orthogonalize(g)
    _check(o, g)
    assert torch.equal(o, F.orthogonalize(g))
    _check(F.orthogonalize(g[-1]), g[-1])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("mats", [[(64, 800)], [(40, 90), (16, 1000), (70, 9)],
                                  [(128, 384), (200, 130), (33, 65)]])
def test_muon_step(device, mats):
    """w <- (1 - lr wd) w - lr gain O(g + mu mom). U is off by 6 roundings at
    most, which the 8 times cover; w takes four operations."""
    lr, mu, wd, scale = 0.02, 0.95, 0.1, 0.5
    views, total = [], 8
    for m, n in mats:
        views.append((total, m, n))
        total += (m * n + 7) // 8 * 8 + 8
    gen = torch.Generator().manual_seed(2)
    st = {k: torch.randn(total, generator=gen) * s for k, s in
          (("master", 0.05), ("grad", 1e-3), ("mom", 4e-3))}
    old = {k: v.double() for k, v in st.items()}
    st = {k: v.to(device) for k, v in st.items()}
    F.muon_step(F.MuonPlan(views, total, device), *st.values(),
                st["master"].bfloat16(), lr=lr, mu=mu, wd=wd, gscale=scale)
    norm = torch.linalg.matrix_norm
    for off, m, n in views:
        sl = slice(off, off + m * n)
        g = old["grad"][sl] * scale
        u = (g + mu * (mu * old["mom"][sl] + g)).view(m, n)
        o = _steps(u, torch.float64)
        yard = norm(_steps(u, torch.float32).double() - o)
        assert yard <= 1800 * math.sqrt(max(m, n)) * U * norm(o)
        step = lr * max(1.0, m / n) ** 0.5
        w = (1 - lr * wd) * old["master"][sl].view(m, n)
        err = st["master"][sl].double().cpu().view(m, n) - (w - step * o)
        tol = step * (8 * yard + 512 * U * norm(o)) + 4 * U * (norm(w)
                                                              + step * norm(o))
        assert norm(err) <= tol


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", [(64, 640), (24, 1000), (128, 640),
                                   (640, 128), (300, 300)])
@pytest.mark.parametrize("small", [1.0, 1e-2, 1e-4, 1e-6, 1e-8])
def test_rows_far_below_the_norm(device, shape, small):
    """Half of the short side's rows are scaled down. What fp32 keeps relative
    to a row, two fp16 halves keep down to half a step of the lower half's
    scale: 2^-25 / 2^14 = 2^-39 for X and A, whose scale is 2^14, and 2^-38 for
    C. On n columns and m rows, a step takes from a row sqrt(n) 2^-39 through X,
    and sqrt(m) |X| <= 1.21 sqrt(m) times what an element of C is off by: its
    own 2^-38, |b| 2^-39 and 2 |c| 1.21^2 2^-39 through A. That is below
    (sqrt(n) + 16 sqrt(m)) 2^-39, and what a row loses in one step grows by
    a in each later one, 1 + a + ... + a^4 = 200."""
    gen = torch.Generator().manual_seed(4)
    m, n = shape
    g = torch.randn(m, n, generator=gen)
    tall = m > n
    (g.T if tall else g)[::2] *= small
    got = F.orthogonalize(g.to(device)).double().cpu()
    ref = _steps(g, torch.float64)
    yard = (_steps(g, torch.float32).double() - ref)
    got, ref, yard = (t.T if tall else t for t in (got, ref, yard))
    m, n = ref.shape
    size = ref.norm(dim=1)
    tol = 8 * yard.norm(dim=1) + 512 * U * size \
        + 200 * (math.sqrt(n) + 16 * math.sqrt(m)) * 2.0 ** -39
    err = (got - ref).norm(dim=1)
    assert bool((err <= tol).all()), f"off by {(err / tol).max():.2f} tolerances"
