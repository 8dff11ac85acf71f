"""Op-level functional API: HIP kernels on GPU, plain-PyTorch fp32 reference
on CPU.

Dispatch rule (the build contract): a CUDA/HIP tensor MUST run the in-tree
gfx950 kernel — ``require_ext()`` raises rather than silently falling back to
eager PyTorch; CPU tensors run the reference implementation (which is also
what GPU numerics tests compare against). Shapes the native GEMM doesn't
cover fall back to torch.matmul (= rocBLAS, a plain library GEMM) — only the
cold path ever takes that branch.

Activation layout is NHWC everywhere (SURVEY §2.9 + conv_pool.hip header).
"""
from __future__ import annotations

import math
import os
from typing import Optional, Tuple

import torch

from ._ext import require_ext


def _is_gpu(t: torch.Tensor) -> bool:
    return t.is_cuda


# --------------------------------------------------------------------- GEMM
def gemm(A: torch.Tensor, B: torch.Tensor, *, ta: bool = False, tb: bool = False,
         bias: Optional[torch.Tensor] = None, relu: bool = False,
         out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
         splits: int = 1, stats: Optional[torch.Tensor] = None,
         addend: Optional[torch.Tensor] = None) -> torch.Tensor:
    """C[M,N] = op(A) @ op(B) (+bias) (+relu). bf16 inputs, fp32 accumulate.

    op(A) = A.T if ta (A stored [K,M]); op(B) = B.T if tb (B stored [N,K]).
    splits > 1 uses the split-K fp32-atomic path (out must be fp32, zeroed
    here).
    """
    M = A.shape[1] if ta else A.shape[0]
    N = B.shape[0] if tb else B.shape[1]
    K = A.shape[0] if ta else A.shape[1]
    dtype = out_dtype or (torch.float32 if splits > 1 else A.dtype)
    if out is None:
        out = torch.empty((M, N), device=A.device, dtype=dtype)
    if _is_gpu(A):
        # PLAIN (F,T) GEMMs with a large N*K panel go to rocBLAS — the
        # sanctioned "plain library GEMM" case (no fused epilogue to carry).
        # Measured crossover on ResNet/MNIST dX shapes (benchmarks/
        # rn_gemm_ab.py): rocBLAS wins 1.2-1.9x above N*K ~= 256k
        # ((1024,256) 0.59, (512,2048) 0.57, (4608,512) 0.61) while the
        # native tile kernel wins below it ((1152,128) 1.02, (64,64) 1.93).
        # Every fused GEMM (bias/ReLU/BN-stats/addend/split-K) stays native.
        if (not ta and tb and bias is None and not relu and stats is None
                and addend is None and splits == 1
                and A.dtype == torch.bfloat16 and out.dtype == torch.bfloat16
                and N * K >= 256 * 1024
                and os.environ.get("LO_PLAIN_ROCBLAS", "1") == "1"):
            torch.matmul(A, B.t(), out=out)
            return out
        lo = require_ext()
        if splits > 1:
            out.zero_()
        if stats is not None:
            stats.zero_()  # epilogue accumulates per-column sum/sumsq
        ok = lo.gemm(A, B, out, bias, ta, tb, 1 if relu else 0, splits,
                     stats.view(-1) if stats is not None else None, addend)
        if ok:
            return out
        # cold-path shapes: plain library GEMM (rocBLAS via torch.matmul)
    a = (A.transpose(0, 1) if ta else A).float()
    b = (B.transpose(0, 1) if tb else B).float()
    c = a @ b
    if bias is not None:
        c = c + bias.float()
    if relu:
        c = torch.relu(c)
    if addend is not None:
        c = c + addend.reshape(c.shape).float()
    out.copy_(c.to(out.dtype))
    return out


# ------------------------------------------------------------------- im2col
def im2col(x: torch.Tensor, kh: int, kw: int, sh: int, sw: int, ph: int, pw: int,
           kpad: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """NHWC x [B,H,W,C] -> col [B*OH*OW, kpad] with row layout (kh, kw, c),
    zero-padded to kpad columns."""
    B, H, W, C = x.shape
    OH = (H + 2 * ph - kh) // sh + 1
    OW = (W + 2 * pw - kw) // sw + 1
    K = kh * kw * C
    assert kpad >= K and kpad % 8 == 0
    if out is None:
        out = torch.zeros((B * OH * OW, kpad), device=x.device, dtype=x.dtype)
    if _is_gpu(x):
        lo = require_ext()
        lo.im2col(x, kh, kw, sh, sw, ph, pw, kpad, out)
        return out
    # reference: unfold on NCHW then reorder (c,kh,kw) -> (kh,kw,c)
    xn = x.permute(0, 3, 1, 2).float()  # NCHW
    cols = torch.nn.functional.unfold(xn, (kh, kw), padding=(ph, pw),
                                      stride=(sh, sw))  # [B, C*kh*kw, L]
    cols = cols.reshape(B, C, kh * kw, -1).permute(0, 3, 2, 1)  # [B,L,khkw,C]
    cols = cols.reshape(B * OH * OW, K)
    out[:, :K] = cols.to(out.dtype)
    out[:, K:] = 0
    return out


def col2im(dcol: torch.Tensor, B: int, H: int, W: int, C: int, kh: int, kw: int,
           sh: int, sw: int, ph: int, pw: int,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gather-form col2im for any stride: dcol [B*OH*OW, kpad] -> dx [B,H,W,C]."""
    OH = (H + 2 * ph - kh) // sh + 1
    OW = (W + 2 * pw - kw) // sw + 1
    if out is None:
        out = torch.empty((B, H, W, C), device=dcol.device, dtype=dcol.dtype)
    if _is_gpu(dcol):
        lo = require_ext()
        lo.col2im(dcol, B, H, W, C, kh, kw, sh, sw, ph, pw, out)
        return out
    K = kh * kw * C
    cols = dcol[:, :K].float().reshape(B, OH * OW, kh * kw, C)
    cols = cols.permute(0, 3, 2, 1).reshape(B, C * kh * kw, OH * OW)
    xn = torch.nn.functional.fold(cols, (H, W), (kh, kw), padding=(ph, pw),
                                  stride=(sh, sw))
    out.copy_(xn.permute(0, 2, 3, 1).to(out.dtype))
    return out


def conv2d_fwd_small(x: torch.Tensor, w: torch.Tensor, kh: int, kw: int,
                     sh: int, sw: int, ph: int, pw: int,
                     bias: Optional[torch.Tensor] = None, relu: bool = False,
                     out: Optional[torch.Tensor] = None) -> bool:
    """GPU-only small-image fused conv forward (x image LDS-resident, w
    tiles double-buffered): pure read-x + write-y traffic.  Returns False
    when not eligible (H*W*(2C+16)+8K > 56KB LDS, outC > 64, ...)."""
    if not x.is_cuda:
        return False
    lo = require_ext()
    return bool(lo.conv_fwd_small(x, w, bias, out, kh, kw, sh, sw, ph, pw,
                                  relu))


def conv1d_fwd(x: torch.Tensor, w: torch.Tensor, kh: int, ph: int,
               bias: Optional[torch.Tensor] = None, relu: bool = False,
               out: Optional[torch.Tensor] = None) -> bool:
    """GPU-only 1-D (W==1, KW==1, stride 1) conv forward: h-tiled x window
    in LDS, outC in 64-wide slices.  False when not eligible."""
    if not x.is_cuda:
        return False
    lo = require_ext()
    return bool(lo.conv1d_fwd(x, w, bias, out, kh, ph, relu))


def conv1d_dx(dy2: torch.Tensor, wt: torch.Tensor, kh: int, ph: int,
              out: torch.Tensor, accumulate: bool = False) -> bool:
    """GPU-only 1-D conv dX: h-tiled LDS fp32 accumulator, non-atomic RMW
    scatter (no dcol matrix).  ``accumulate`` adds into ``out`` instead of
    overwriting (fuses the TextCNN branch-grad sum).  False when not
    eligible."""
    if not dy2.is_cuda:
        return False
    lo = require_ext()
    return bool(lo.conv1d_dx(dy2, wt, out, kh, ph, accumulate))


def conv2d_dw_small(dy2: torch.Tensor, x: torch.Tensor, gw: torch.Tensor,
                    kh: int, kw: int, sh: int, sw: int, ph: int, pw: int) -> bool:
    """GPU-only small-image multi-channel conv weight grad: x + transposed
    dy LDS-resident per image, register-accumulated kpad chunks — built to
    kill the gather-GEMM's per-kpad-tile dY re-streaming (3.5 GB on MNIST
    conv2). Measured r2: ~1% SLOWER than the gather GEMM end-to-end (8.05
    vs 8.13 M samples/s) — the per-element scalar LDS gathers of the
    B operand pay in bank conflicts what the halved dY traffic saves — so
    it is OFF by default (LO_DW_SMALL=1 enables; kernel + numerics tests
    kept as the documented alternative).  gw fp32, zeroed inside."""
    if not dy2.is_cuda:
        return False
    import os
    if os.environ.get("LO_DW_SMALL", "0") != "1":
        return False
    lo = require_ext()
    return bool(lo.conv_dw_small(dy2, x, gw, kh, kw, sh, sw, ph, pw))


def conv2d_dw_c1(dy2: torch.Tensor, x: torch.Tensor, gw: torch.Tensor,
                 kh: int, kw: int, sh: int, sw: int, ph: int, pw: int) -> bool:
    """GPU-only C=1 conv weight grad (dY^T @ im2col(x)) with x images
    LDS-resident — no col matrix, no split-K pass structure.  gw fp32,
    zeroed inside.  Returns False when not eligible (outC > 32, ...)."""
    if not dy2.is_cuda:
        return False
    lo = require_ext()
    return bool(lo.conv_dw_c1(dy2, x, gw, kh, kw, sh, sw, ph, pw))


def conv2d_dx_fused(dy2: torch.Tensor, wt: torch.Tensor, B: int, H: int,
                    W: int, C: int, kh: int, kw: int, sh: int, sw: int,
                    ph: int, pw: int, out: torch.Tensor) -> bool:
    """GPU-only fused conv dX: dcol = dy2 @ wt^T computed per image with MFMA
    and scattered straight into an LDS fp32 dx accumulator — no dcol matrix
    (replaces gemm-NT + col2im).  wt is the [kpad, outC] transposed weight
    mirror.  Returns False when the shape is not eligible (whole-image dx
    must fit LDS: H*W*C*4 <= 48 KB, C%16==0, outC <= 64) — caller falls back."""
    if not dy2.is_cuda:
        return False
    lo = require_ext()
    return bool(lo.conv_dx(dy2, wt, out, kh, kw, sh, sw, ph, pw))


# ------------------------------------------------------------------ maxpool
def maxpool2d(x: torch.Tensor, kh: int, kw: int, sh: int, sw: int,
              ph: int = 0, pw: int = 0,
              relu_mask: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """NHWC maxpool (zero-pad treated as -inf); returns (out, idx u8 of
    kh*KW+kw argmax). ``relu_mask``: positions whose max is <= 0 get
    sentinel idx 255, folding the upstream conv's ReLU backward into the
    index — the pool BACKWARD then needs no relu_y stream (that stream was
    ~40% of the pool-bwd traffic on MNIST)."""
    if _is_gpu(x):
        lo = require_ext()
        out, idx = lo.maxpool_fwd(x, kh, kw, sh, sw, ph, pw,
                                  relu_sentinel=relu_mask)
        return out, idx
    B, H, W, C = x.shape
    OH = (H + 2 * ph - kh) // sh + 1
    OW = (W + 2 * pw - kw) // sw + 1
    xn = x.permute(0, 3, 1, 2).float()
    out_n, ind = torch.nn.functional.max_pool2d(xn, (kh, kw), (sh, sw),
                                                padding=(ph, pw),
                                                return_indices=True)
    out = out_n.permute(0, 2, 3, 1).to(x.dtype)
    # flat NCHW index -> (kh,kw) offset index
    hh = (ind // W)
    ww = (ind % W)
    oh = torch.arange(OH, device=x.device).view(1, 1, OH, 1)
    ow = torch.arange(OW, device=x.device).view(1, 1, 1, OW)
    rel = (hh - (oh * sh - ph)) * kw + (ww - (ow * sw - pw))
    idx = rel.permute(0, 2, 3, 1).to(torch.uint8).contiguous()
    if relu_mask:
        idx[out <= 0] = 255
    return out, idx


def maxpool2d_bwd(dy: torch.Tensor, idx: torch.Tensor, H: int, W: int,
                  kh: int, kw: int, sh: int, sw: int, ph: int = 0, pw: int = 0,
                  out: Optional[torch.Tensor] = None,
                  relu_y: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``relu_y`` (the pool input = upstream conv's ReLU output, same
    [B,H,W,C]) fuses that conv's ReLU backward: dx is zeroed where
    relu_y <= 0, replacing a separate relu_bwd pass."""
    B, OH, OW, C = dy.shape
    if out is None:
        out = torch.empty((B, H, W, C), device=dy.device, dtype=dy.dtype)
    if _is_gpu(dy):
        lo = require_ext()
        lo.maxpool_bwd(dy, idx, H, W, kh, kw, sh, sw, ph, pw, out, relu_y)
        return out
    dx = torch.zeros((B, H, W, C), dtype=torch.float32)
    rel = idx.long()
    valid = rel != 255                 # 255 = fused-ReLU sentinel (no grad)
    rel = torch.where(valid, rel, torch.zeros_like(rel))
    khh, kww = rel // kw, rel % kw
    oh = torch.arange(OH).view(1, OH, 1, 1)
    ow = torch.arange(OW).view(1, 1, OW, 1)
    hsrc = oh * sh + khh - ph
    wsrc = ow * sw + kww - pw
    b = torch.arange(B).view(B, 1, 1, 1).expand_as(rel)
    c = torch.arange(C).view(1, 1, 1, C).expand_as(rel)
    src = torch.where(valid, dy.float(), torch.zeros_like(dy, dtype=torch.float32))
    dx.index_put_((b.reshape(-1), hsrc.reshape(-1), wsrc.reshape(-1),
                   c.reshape(-1)), src.reshape(-1), accumulate=True)
    if relu_y is not None:
        dx = dx * (relu_y.float() > 0)
    out.copy_(dx.to(out.dtype))
    return out


# -------------------------------------------------------------- activations
def relu_bwd(dy: torch.Tensor, y: torch.Tensor,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    if out is None:
        out = torch.empty_like(dy)
    if _is_gpu(dy):
        lo = require_ext()
        lo.relu_bwd(dy.contiguous().view(-1), y.contiguous().view(-1),
                    out.view(-1))
        return out
    out.copy_((dy.float() * (y.float() > 0)).to(out.dtype))
    return out


# ---------------------------------------------------------------- optimizer
def sgd_step(master: torch.Tensor, grad: torch.Tensor, mom: torch.Tensor,
             mirror: torch.Tensor, lr: float, mu: float, wd: float,
             gscale: float = 1.0) -> None:
    if _is_gpu(master):
        lo = require_ext()
        lo.sgd_step(master, grad, mom, mirror, lr, mu, wd, gscale)
        return
    g = grad * gscale + wd * master
    mom.mul_(mu).add_(g)
    master.add_(mom, alpha=-lr)
    mirror.copy_(master.to(mirror.dtype))


def adam_step(master: torch.Tensor, grad: torch.Tensor, m1: torch.Tensor,
              m2: torch.Tensor, mirror: torch.Tensor, lr: float, b1: float,
              b2: float, eps: float, wd: float, step,
              gscale: float = 1.0) -> None:
    """``step``: int on CPU, or an int32 device scalar tensor on GPU (read
    on device -- hipGraph-capture-safe bias correction)."""
    if _is_gpu(master):
        lo = require_ext()
        if not torch.is_tensor(step):
            step = torch.tensor([int(step)], dtype=torch.int32,
                                device=master.device)
        lo.adam_step(master, grad, m1, m2, mirror, step, lr, b1, b2, eps, wd,
                     gscale)
        return
    t = int(step.item()) if torch.is_tensor(step) else int(step)
    c1 = 1.0 / (1.0 - b1 ** t)
    c2 = 1.0 / (1.0 - b2 ** t)
    g = grad * gscale + wd * master
    m1.mul_(b1).add_(g, alpha=1 - b1)
    m2.mul_(b2).addcmul_(g, g, value=1 - b2)
    master.addcdiv_(m1 * c1, (m2 * c2).sqrt() + eps, value=-lr)
    mirror.copy_(master.to(mirror.dtype))


class AdamRanges:
    """Parts of a flat arena, (start, end) pairs of multiples of 8 elements,
    for ``adam_ranges``."""

    def __init__(self, ranges, numel: int, device) -> None:
        self.ranges = [(int(a), int(b)) for a, b in ranges]
        for a, b in self.ranges:
            if not 0 <= a < b <= numel or a % 8 or b % 8:
                raise ValueError("ranges must be multiples of 8 within the "
                                 "arena")
        ordered = sorted(self.ranges)
        if any(a[1] > b[0] for a, b in zip(ordered, ordered[1:])):
            raise ValueError("ranges must not overlap")
        self.numel = int(numel)
        self.longest = max((b - a for a, b in self.ranges), default=0)
        self._table = torch.tensor(self.ranges, dtype=torch.int64,
                                   device=device).view(-1, 2)


def adam_ranges(ranges: AdamRanges, master: torch.Tensor, grad: torch.Tensor,
                m1: torch.Tensor, m2: torch.Tensor, mirror: torch.Tensor,
                lr: float, b1: float, b2: float, eps: float, wd: float, step,
                gscale: float = 1.0) -> None:
    """``adam_step`` on some ranges of the arena, in one launch."""
    if ranges.numel != master.numel():
        raise RuntimeError(f"the ranges are for {ranges.numel} elements")
    if not _is_gpu(master):
        _check_arena(master, grad, m1, m2, mirror)
    if _is_gpu(master):
        if not torch.is_tensor(step):
            step = torch.tensor([int(step)], dtype=torch.int32,
                                device=master.device)
        require_ext().adam_ranges(master, grad, m1, m2, mirror, step,
                                  ranges._table, ranges.longest, lr, b1, b2,
                                  eps, wd, gscale)
        return
    for a, b in ranges.ranges:
        adam_step(master[a:b], grad[a:b], m1[a:b], m2[a:b], mirror[a:b], lr,
                  b1, b2, eps, wd, step, gscale)


def _check_arena(*tensors) -> None:
    # the CPU path refuses what the kernels' bindings refuse
    if any(t.numel() != tensors[0].numel() for t in tensors):
        raise RuntimeError("the arena's tensors must match")
    for i, a in enumerate(tensors):
        if any(_touches(a, b) for b in tensors[:i]):
            raise RuntimeError("the arena's tensors must not share memory")


# ------------------------------------------------- Newton-Schulz and Muon
# the quintic of the published Muon optimizer (Jordan et al., 2024): five steps
# bring singular values from 0.002 up to between 0.68 and 1.21, the steepest
# start at the price of not settling at 1
NS_COEFFS = (3.4445, -4.7750, 2.0315)
NS_SIDE = 1 << 20       # the longest side that a matrix may have


def _ns_coeffs(steps: int, coeffs, eps: float) -> list:
    """[a, b, c] per step, flat, from one triple or one triple per step."""
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    if int(steps) != steps or not 1 <= steps <= 100:
        raise ValueError("Newton-Schulz takes 1 to 100 steps")
    rows = [coeffs] * int(steps) if len(coeffs) == 3 and not hasattr(
        coeffs[0], "__len__") else list(coeffs)
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise ValueError("coeffs: one (a, b, c), or one for each step")
    return [float(v) for r in rows for v in r]


def _ns_bounds(flat: list) -> None:
    """Refuses for the CPU path the coefficients that the bindings refuse
    (newton_schulz_plan.h), whose powers of two would leave fp32's range."""
    top = 1.001         # the singular values' bound, before and after a step
    for a, b, c in zip(*[iter(flat)] * 3):
        if not all(abs(v) <= torch.finfo(torch.float32).max for v in (a, b, c)):
            raise ValueError("coeffs must be finite in fp32")
        if 0 < top < 2.0 ** -20:
            raise ValueError("these coefficients let the singular values fall "
                             "below 2^-20 before a step")
        # |a + b q + c q^2| is largest at an end or where its slope is zero, and
        # sqrt(q) times it at the end or where a + 3 b q + 5 c q^2 = 0
        q, disc = [0.0, top * top], 9 * b * b - 20 * a * c
        if c:
            q.append(-b / (2 * c))
        if c and disc >= 0:
            q += [(-3 * b + r * math.sqrt(disc)) / (10 * c) for r in (1, -1)]
        elif not c and b:
            q.append(-a / (3 * b))
        q = [v for v in q if 0 <= v <= top * top]
        poly = [abs(a + b * v + c * v * v) for v in q]
        most = max(math.sqrt(v) * p for v, p in zip(q, poly))
        if most >= 2 ** 20 or max(poly) >= 2 ** 40:
            raise ValueError("these coefficients let the singular values "
                             "grow past 2^20, or a step's polynomial past 2^40")
        if 0 < max(poly) < 2.0 ** -40:
            raise ValueError("these coefficients make a step's polynomial "
                             "fall below 2^-40")
        top = most * 1.001


def _newton_schulz_ref(x: torch.Tensor, flat: list, eps: float) -> torch.Tensor:
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    x = x.double()
    norm = x.square().sum((-2, -1), keepdim=True).sqrt() + eps
    x = (x / norm.where(norm != 0, 1.0)).float()
    for i in range(0, len(flat), 3):
        a, b, c = flat[i:i + 3]
        gram = x @ x.transpose(-2, -1)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-2, -1) if tall else x


def orthogonalize(g: torch.Tensor, steps: int = 5, coeffs=NS_COEFFS,
                  eps: float = 1e-7,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """G with its singular values brought towards one, by Newton-Schulz steps
    X <- a X + (b A + c A^2) X, A = X X^T, from X = G / (|G|_F + eps). With
    NS_COEFFS, five steps leave them between 0.68 and 1.21, but for those below
    0.002 of the norm; steps that settle at one, as (1.5, -0.5, 0), end at the
    nearest matrix with orthonormal rows (or columns, if tall).

    g [m, n] or a batch [..., m, n] in bf16, fp16 or fp32; rounded once to
    ``out``, of g's shape and type (it may be g). The error is that of fp32
    steps in the norm of the whole matrix; a GPU keeps values down to 2^-38 of
    it, so rows below 1e-4 of the others lose digits of their own that fp32
    would keep (1e-6: relative error 2e-4).

    ``coeffs``: (a, b, c), or a triple for each step. Refused are those that
    can bring a singular value past 2^20 or, before a step, below 2^-20, and
    polynomials a + b q + c q^2 that stay below 2^-40. A zero matrix stays zero.
    A view that is not contiguous is copied first. The same call gives the same
    bits; batches of other sizes may sum in another order."""
    flat = _ns_coeffs(steps, coeffs, eps)
    if g.dim() < 2:
        raise ValueError("g must be a matrix or a batch of them")
    if g.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError("g must be bf16, fp16 or fp32")
    if max(g.shape[-2:]) > NS_SIDE:
        raise ValueError(f"a matrix's sides end at {NS_SIDE}")
    if out is None:
        out = torch.empty_like(g, memory_format=torch.contiguous_format)
    if out.shape != g.shape or out.dtype != g.dtype or out.device != g.device \
            or not out.is_contiguous():
        raise ValueError("out must be contiguous and of g's shape, type and "
                         "device")
    if g.is_contiguous() and not _apart(out.view(1, -1), g.view(1, -1)):
        raise ValueError("out may be g, but not overlap it in part")
    if _is_gpu(g):
        three = (-1 if g.numel() else 0, g.shape[-2], g.shape[-1])
        require_ext().orthogonalize(g.contiguous().view(three),
                                    out.view(three), flat, eps)
        return out
    _ns_bounds(flat)
    if g.numel():
        out.copy_(_newton_schulz_ref(g.contiguous().float(), flat, eps))
    return out


class MuonPlan:
    """What ``muon_step`` keeps between steps for the weight matrices of one
    flat arena of ``numel`` elements: ``views`` lists them as (offset, rows,
    cols), offsets being multiples of 8 as ParamArena's are. On a GPU it owns
    the kernels' tables and their workspace (about 8 bytes an element for wide
    matrices), so steps that share a plan have to be ordered, like steps that
    share a momentum, and the plan has to outlive graphs that captured them.

    ``sides`` lists the matrices' own (rows, cols) where the stored ones count
    rows or columns of padding, which hold zeros: the factor on the learning
    rate goes by the own sides, and zeros change nothing else."""

    def __init__(self, views, numel: int, device, sides=None) -> None:
        self.views = [tuple(int(v) for v in t) for t in views]
        self.numel = int(numel)
        self.device = torch.device(device)
        if any(len(t) != 3 for t in self.views) or not self.views:
            raise ValueError("views: (offset, rows, cols) for each matrix")
        end = 0
        for off, m, n in sorted(self.views):
            if off < end or off % 8 or m < 1 or n < 1:
                raise ValueError("matrices must start on a multiple of 8 "
                                 "elements and not overlap")
            if max(m, n) > NS_SIDE:
                raise ValueError(f"a matrix's sides end at {NS_SIDE}")
            end = off + m * n
        if end > self.numel:
            raise ValueError("a matrix ends outside the arena")
        self.sides = [t[1:] for t in self.views] if sides is None else \
            [tuple(int(v) for v in t) for t in sides]
        if len(self.sides) != len(self.views) or any(
                len(s) != 2 or not (1 <= s[0] <= m and 1 <= s[1] <= n)
                for s, (_, m, n) in zip(self.sides, self.views)):
            raise ValueError("sides: each matrix's own (rows, cols), at most "
                             "the stored ones")
        self.gains = [math.sqrt(max(1.0, m / n)) for m, n in self.sides]
        self._native = None
        if self.device.type == "cuda":
            dev = self.device if self.device.index is not None else \
                torch.device("cuda", torch.cuda.current_device())
            order = sorted(range(len(self.views)), key=self.views.__getitem__)
            self._native = require_ext().MuonPlan(
                [list(self.views[i]) for i in order],
                [self.gains[i] for i in order], self.numel, str(dev))

    def __reduce__(self):   # copies and pickles are plans of their own
        return MuonPlan, (self.views, self.numel, str(self.device), self.sides)


def muon_step(plan: MuonPlan, master: torch.Tensor, grad: torch.Tensor,
              mom: torch.Tensor, mirror: torch.Tensor, lr: float,
              mu: float = 0.95, wd: float = 0.0, gscale: float = 1.0,
              nesterov: bool = True, steps: int = 5, coeffs=NS_COEFFS,
              eps: float = 1e-7) -> None:
    """One Muon step of the plan's matrices, in place on flat fp32 master,
    grad and momentum and the bf16 mirror:

        mom <- mu mom + gscale g;  U = gscale g + mu mom (nesterov) or mom
        w <- (1 - lr wd) w - lr sqrt(max(1, rows / cols)) orthogonalize(U)

    where rows and cols are the plan's ``sides``. Elements outside the matrices
    stay as they are. Every rank that starts from the same values ends with the
    same values."""
    flat = _ns_coeffs(steps, coeffs, eps)
    if plan._native is not None:
        plan._native.step(master, grad, mom, mirror, lr, mu, wd, gscale,
                          nesterov, flat, eps)
        return
    for t in (master, grad, mom, mirror):
        if t.numel() != plan.numel or t.is_cuda:
            raise RuntimeError(f"the plan is for {plan.numel} elements on "
                               f"{plan.device}")
    _check_arena(master, grad, mom, mirror)
    _ns_bounds(flat)
    for (off, m, n), gain in zip(plan.views, plan.gains):
        sl = slice(off, off + m * n)
        g = grad[sl] * gscale
        mom[sl].mul_(mu).add_(g)
        u = g + mu * mom[sl] if nesterov else mom[sl]
        o = _newton_schulz_ref(u.view(m, n), flat, eps).reshape(-1)
        master[sl].mul_(1.0 - lr * wd).add_(o, alpha=-lr * gain)
        mirror[sl] = master[sl].to(mirror.dtype)


# --------------------------------------------------------------- reductions
def colsum(dy: torch.Tensor, out: Optional[torch.Tensor] = None,
           mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``mask``: optional u8 array (same shape); elements with value 255 are
    EXCLUDED (the maxpool ReLU-sentinel) — lets bias grads sum the small
    pool-level grad instead of the scattered full-resolution one."""
    if out is None:
        out = torch.empty(dy.shape[1], device=dy.device, dtype=torch.float32)
    if _is_gpu(dy):
        lo = require_ext()
        lo.colsum(dy, out, mask)
        return out
    d = dy.float()
    if mask is not None:
        d = torch.where(torch.as_tensor(mask).view(dy.shape) != 255, d,
                        torch.zeros((), dtype=d.dtype))
    out.copy_(d.sum(0))
    return out


def argmax_rows(x: torch.Tensor, cvalid: Optional[int] = None) -> torch.Tensor:
    cvalid = cvalid or x.shape[1]
    if _is_gpu(x):
        lo = require_ext()
        return lo.argmax_rows(x, cvalid)
    return x[:, :cvalid].float().argmax(1).to(torch.int32)


def accuracy_count(pred: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    if _is_gpu(pred):
        lo = require_ext()
        return lo.accuracy_count(pred, labels)
    return (pred.long() == labels).sum().to(torch.int32).reshape(1)


# --------------------------------------------------------------- softmax-CE
def softmax_ce(logits: torch.Tensor, labels: torch.Tensor,
               dlogits: Optional[torch.Tensor] = None,
               loss_sum: Optional[torch.Tensor] = None,
               correct: Optional[torch.Tensor] = None,
               cvalid: Optional[int] = None, gscale: float = 1.0):
    """Fused fwd+bwd: writes dlogits; accumulates loss_sum (fp32[1]) and
    correct (int32[1]) in place. Returns (dlogits, loss_sum, correct)."""
    M, C = logits.shape
    cvalid = cvalid or C
    if dlogits is None:
        dlogits = torch.empty_like(logits)
    if loss_sum is None:
        loss_sum = torch.zeros(1, device=logits.device, dtype=torch.float32)
    if correct is None:
        correct = torch.zeros(1, device=logits.device, dtype=torch.int32)
    if _is_gpu(logits):
        lo = require_ext()
        lo.softmax_ce(logits, labels, dlogits, loss_sum, correct, cvalid, gscale)
        return dlogits, loss_sum, correct
    lg = logits[:, :cvalid].float()
    p = torch.softmax(lg, dim=1)
    loss = torch.nn.functional.cross_entropy(lg, labels, reduction="sum")
    onehot = torch.nn.functional.one_hot(labels, cvalid).float()
    d = (p - onehot) * gscale
    dlogits.zero_()
    dlogits[:, :cvalid] = d.to(dlogits.dtype)
    loss_sum += loss
    correct += (lg.argmax(1) == labels).sum().to(torch.int32)
    return dlogits, loss_sum, correct


# ---------------------------------------------------------------- embedding
def embedding(ids: torch.Tensor, table: torch.Tensor,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gather rows: out[..., :] = table[ids[...], :] (bf16)."""
    dim = table.shape[1]
    if out is None:
        out = torch.empty(*ids.shape, dim, device=table.device, dtype=table.dtype)
    if _is_gpu(table):
        lo = require_ext()
        lo.embedding_fwd(ids.contiguous(), table, out.view(-1, dim))
        return out
    out.copy_(table[ids])
    return out


def embedding_bwd(ids: torch.Tensor, dy: torch.Tensor,
                  gtable: torch.Tensor) -> None:
    """Scatter-add: gtable[ids[...], :] += dy (fp32 accumulate). Caller zeros
    gtable (the grad arena is fully rewritten each step)."""
    dim = gtable.shape[1]
    if _is_gpu(gtable):
        lo = require_ext()
        lo.embedding_bwd(ids.contiguous(), dy.contiguous().view(-1, dim), gtable)
        return
    gtable.index_add_(0, ids.reshape(-1), dy.float().reshape(-1, dim))


# --------------------------------------------------------------- batchnorm
def bn_fwd_train(x2d: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor,
                 eps: float, out: torch.Tensor, mean: torch.Tensor,
                 invstd: torch.Tensor, scratch: torch.Tensor,
                 relu: bool = True, stats_ready: bool = False,
                 residual: Optional[torch.Tensor] = None,
                 running: Optional[tuple] = None,
                 momentum: float = 0.0) -> None:
    """Training-mode BN over [M, C] (+fused ReLU). Writes out (bf16), mean,
    invstd (fp32 [C]); ``scratch`` is a [2, C] fp32 workspace (sum/sumsq).
    ``stats_ready``: scratch was already filled by the producing GEMM's fused
    epilogue — skip the bn_stats pass. ``running`` = (running_mean,
    running_var): on GPU the EMA update fuses into the same finalize kernel
    (one launch instead of ~12 torch elementwise ops per BN per step)."""
    M, C = x2d.shape
    if _is_gpu(x2d):
        lo = require_ext()
        if not stats_ready:
            lo.bn_stats(x2d, scratch[0], scratch[1])
        if running is not None:
            lo.bn_finalize_stats(scratch, mean, invstd, M, running[0],
                                 running[1], momentum, eps)
        else:
            lo.bn_finalize_stats(scratch, mean, invstd, M, eps=eps)
        lo.bn_fwd(x2d, out, mean, invstd, gamma, beta, relu,
                  residual.reshape(M, C) if residual is not None else None)
        return
    xf = x2d.float()
    mean.copy_(xf.mean(0))
    invstd.copy_((xf.var(0, unbiased=False) + eps).rsqrt())
    y = (xf - mean) * invstd * gamma + beta
    if residual is not None:
        y = y + residual.reshape(M, C).float()
    if relu:
        y = torch.relu(y)
    out.copy_(y.to(out.dtype))


def bn_fwd_eval(x2d: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor,
                running_mean: torch.Tensor, running_var: torch.Tensor,
                eps: float, out: torch.Tensor, relu: bool = True,
                residual: Optional[torch.Tensor] = None) -> None:
    invstd = (running_var + eps).rsqrt()
    if _is_gpu(x2d):
        lo = require_ext()
        lo.bn_fwd(x2d, out, running_mean.contiguous(), invstd.contiguous(),
                  gamma, beta, relu,
                  residual.reshape(x2d.shape) if residual is not None else None)
        return
    y = (x2d.float() - running_mean) * invstd * gamma + beta
    if residual is not None:
        y = y + residual.reshape(x2d.shape).float()
    if relu:
        y = torch.relu(y)
    out.copy_(y.to(out.dtype))


def bn_bwd(dy2d: torch.Tensor, y2d: torch.Tensor, x2d: torch.Tensor,
           mean: torch.Tensor, invstd: torch.Tensor, gamma: torch.Tensor,
           dgamma: torch.Tensor, dbeta: torch.Tensor, dx: torch.Tensor,
           relu: bool = True) -> None:
    """BN backward (ReLU-fused variant masks dy by y>0). Writes dgamma,
    dbeta (fp32 [C], overwritten) and dx (bf16 [M,C])."""
    M, C = x2d.shape
    if _is_gpu(x2d):
        lo = require_ext()
        lo.bn_bwd_reduce(dy2d, y2d, x2d, mean, invstd, dbeta, dgamma, relu)
        lo.bn_bwd_dx(dy2d, y2d, x2d, dx, mean, invstd, gamma, dbeta, dgamma,
                     relu)
        return
    g = dy2d.float()
    if relu:
        g = g * (y2d.float() > 0)
    xhat = (x2d.float() - mean) * invstd
    dbeta.copy_(g.sum(0))
    dgamma.copy_((g * xhat).sum(0))
    d = gamma * invstd * (g - dbeta / M - xhat * dgamma / M)
    dx.copy_(d.to(dx.dtype))


# --------------------------------------------------------------- layernorm
def layernorm_fwd(x2d: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor,
                  eps: float, out: torch.Tensor,
                  mean: Optional[torch.Tensor] = None,
                  invstd: Optional[torch.Tensor] = None,
                  residual: Optional[torch.Tensor] = None,
                  sum_out: Optional[torch.Tensor] = None) -> None:
    """Layer norm over the rows of x2d [M, C] (bf16, fp16 or fp32, any row
    stride, 1 <= C <= 32768) with fp32 gamma/beta [C]. Writes out (x2d's type)
    and, for training, mean and invstd (fp32 [M]). ``residual`` [M, C] is
    added first; the sum, rounded to x2d's type, is what gets normalised and
    goes to ``sum_out`` (the backward pass's x2d). ``out`` and ``sum_out`` may
    each be one of x2d and the residual, but not a part of one; outputs share
    no memory otherwise."""
    if _is_gpu(x2d):
        require_ext().layernorm_fwd(x2d, gamma, beta, eps, out, mean, invstd,
                                    residual, sum_out)
        return
    _check_layernorm(x2d, (out, residual, sum_out), (gamma, beta),
                     (mean, invstd), (out, sum_out), (gamma, beta),
                     (mean, invstd))
    if (mean is None) != (invstd is None):
        raise RuntimeError("mean and invstd come together")
    if sum_out is not None and residual is None:
        raise RuntimeError("sum_out needs a residual")
    s = x2d
    if residual is not None:
        s = (x2d.float() + residual.float()).to(x2d.dtype)
    xf = s.float()
    mu = xf.mean(1, keepdim=True)
    rstd = ((xf - mu).square().mean(1, keepdim=True) + eps).rsqrt()
    y = ((xf - mu) * rstd * gamma + beta).to(out.dtype)
    if sum_out is not None:
        sum_out.copy_(s)
    out.copy_(y)
    if mean is not None:
        mean.copy_(mu.view(-1))
        invstd.copy_(rstd.view(-1))


def layernorm_bwd(dy2d: torch.Tensor, x2d: torch.Tensor, mean: torch.Tensor,
                  invstd: torch.Tensor, gamma: torch.Tensor,
                  dgamma: torch.Tensor, dbeta: torch.Tensor, dx: torch.Tensor,
                  dskip: Optional[torch.Tensor] = None) -> None:
    """Layer norm backward from what ``layernorm_fwd`` normalised (x2d, or its
    ``sum_out``) and its mean/invstd. Writes dgamma, dbeta (fp32 [C],
    overwritten; the same sums on every run) and dx. ``dskip`` [M, C], the
    gradient that reaches the sum past the norm, is added to dx, which then is
    the gradient of x and of the residual alike. ``dx`` may be dy2d, x2d or
    dskip, but not a part of one; outputs share no memory otherwise."""
    if _is_gpu(x2d):
        require_ext().layernorm_bwd(dy2d, x2d, mean, invstd, gamma, dgamma,
                                    dbeta, dx, dskip)
        return
    _check_layernorm(x2d, (dy2d, dx, dskip), (gamma, dgamma, dbeta),
                     (mean, invstd), (dx,), (gamma, mean, invstd),
                     (dgamma, dbeta))
    g = dy2d.float()
    xhat = (x2d.float() - mean.view(-1, 1)) * invstd.view(-1, 1)
    h = g * gamma
    d = invstd.view(-1, 1) * (h - h.mean(1, keepdim=True)
                              - xhat * (h * xhat).mean(1, keepdim=True))
    if dskip is not None:
        d = d + dskip.float()
    dgamma.copy_((g * xhat).sum(0))
    dbeta.copy_(g.sum(0))
    dx.copy_(d.to(dx.dtype))


def _apart(out: torch.Tensor, x: torch.Tensor) -> bool:
    # out is x, or shares no element with it, or lies beside it in wider rows
    if not out.numel() or out.device != x.device:
        return True
    (rows, cols), size = out.shape, out.element_size()
    lo, li = (t.stride(0) if rows > 1 else cols for t in (out, x))
    a, b = out.data_ptr(), x.data_ptr()
    if (a, lo) == (b, li) or a + ((rows - 1) * lo + cols) * size <= b \
            or b + ((rows - 1) * li + cols) * size <= a:
        return True
    return lo == li and cols * size <= (a - b) % (lo * size) <= (lo - cols) * size


def _touches(t: torch.Tensor, vec: torch.Tensor) -> bool:
    # whether some row of t (cut to its columns) shares memory with vec
    if not t.numel() or not vec.numel() or t.device != vec.device:
        return False
    size = t.element_size()
    row = t.stride(0) * size if t.dim() > 1 and t.shape[0] > 1 else 0
    rows = t.shape[0] if row else 1
    width = (t.shape[1] if t.dim() > 1 else t.numel()) * size
    at, v = t.data_ptr(), vec.data_ptr()
    r = (v - at - width) // row + 1 if row and v - at >= width else 0
    return r < rows and at + r * row < v + vec.numel() * vec.element_size() \
        and at + r * row + width > v


def _check_layernorm(x, rows, vecs, stats, outs, vec_ins, vec_outs) -> None:
    # the CPU path refuses what the kernels' bindings refuse
    if x.dim() != 2 or not 1 <= x.shape[1] <= 32768:
        raise RuntimeError("layer norm takes [rows, 1 to 32768 columns]")
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise RuntimeError("x must be bf16, fp16 or fp32")
    for t in rows:
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype
                              or t.device != x.device):
            raise RuntimeError("activations must have the input's shape, "
                               "type and device")
    if x.shape[1] > 1 and any(t is not None and t.stride(1) != 1
                              for t in (x, *rows)):
        raise RuntimeError("activations must be contiguous along their columns")
    for group, n in ((vecs, x.shape[1]), (stats, x.shape[0])):
        for t in group:
            if t is not None and (t.numel() != n or t.dtype != torch.float32
                                  or t.device != x.device):
                raise RuntimeError(f"statistics and parameters must be fp32 "
                                   f"with {n} values")
    for o in outs:
        if o is not None and o.shape[0] > 1 and o.stride(0) < o.shape[1]:
            raise RuntimeError("an output must not overlap itself")
        for t in (x, *rows):
            if None not in (o, t) and o is not t and not _apart(o, t):
                raise RuntimeError("an output may be an input, but not overlap "
                                   "one in part")
    # pairs of which one is written and one is a vector
    pairs = [(o, v) for o in outs for v in vec_ins]
    for i, v in enumerate(vec_outs):
        pairs += [(t, v) for t in (x, *rows, *vec_ins, *vec_outs[:i])]
    if any(t is not None and v is not None and _touches(t, v)
           for t, v in pairs):
        raise RuntimeError("statistics, parameters and their gradients must "
                           "not share memory with an output")


# ------------------------------------------------------------ residual add
def add_relu(a: torch.Tensor, b: torch.Tensor, out: Optional[torch.Tensor] = None,
             relu: bool = True) -> torch.Tensor:
    if out is None:
        out = torch.empty_like(a)
    if _is_gpu(a):
        lo = require_ext()
        lo.add_relu(a.view(-1), b.view(-1), out.view(-1), relu)
        return out
    z = a.float() + b.float()
    if relu:
        z = torch.relu(z)
    out.copy_(z.to(out.dtype))
    return out


# ------------------------------------------------------ global average pool
def avgpool_global(x: torch.Tensor, out: Optional[torch.Tensor] = None
                   ) -> torch.Tensor:
    """[B,H,W,C] -> [B,C] mean over H*W."""
    B, H, W, C = x.shape
    if out is None:
        out = torch.empty((B, C), device=x.device, dtype=x.dtype)
    if _is_gpu(x):
        lo = require_ext()
        lo.avgpool_global(x, out)
        return out
    out.copy_(x.float().mean((1, 2)).to(out.dtype))
    return out


def avgpool_global_bwd(dy: torch.Tensor, H: int, W: int,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    B, C = dy.shape
    if out is None:
        out = torch.empty((B, H, W, C), device=dy.device, dtype=dy.dtype)
    if _is_gpu(dy):
        lo = require_ext()
        lo.avgpool_global_bwd(dy, out)
        return out
    out.copy_((dy.float() / (H * W)).view(B, 1, 1, C)
              .expand(B, H, W, C).to(out.dtype))
    return out


# ------------------------------------------------------- implicit-GEMM conv
def conv2d_fwd_implicit(x: torch.Tensor, w: torch.Tensor, kh: int, kw: int,
                        sh: int, sw: int, ph: int, pw: int,
                        bias: Optional[torch.Tensor] = None, relu: bool = False,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """GPU-only fused conv forward: y2d[B*OH*OW, outC] = im2col(x) @ w^T
    gathered inside the GEMM staging (no col matrix). w is [outC, kpad]."""
    assert x.is_cuda
    B, H, W, C = x.shape
    OH = (H + 2 * ph - kh) // sh + 1
    OW = (W + 2 * pw - kw) // sw + 1
    if out is None:
        out = torch.empty((B * OH * OW, w.shape[0]), device=x.device,
                          dtype=x.dtype)
    lo = require_ext()
    ok = lo.gemm_conv_fwd(x, w, out, bias, relu, kh, kw, sh, sw, ph, pw)
    if not ok:
        raise RuntimeError("gemm_conv_fwd: no config for this shape")
    return out


def conv2d_dw_implicit(dy2: torch.Tensor, x: torch.Tensor, gw: torch.Tensor,
                       kh: int, kw: int, sh: int, sw: int, ph: int, pw: int,
                       splits: int) -> torch.Tensor:
    """GPU-only fused conv weight grad: gw[outC, kpad] = dY^T @ im2col(x),
    split-K fp32 atomics (gw zeroed here)."""
    assert x.is_cuda
    lo = require_ext()
    gw.zero_()
    ok = lo.gemm_conv_dw(dy2, x, gw, max(splits, 2), kh, kw, sh, sw, ph, pw)
    if not ok:
        # shapes the gather path can't take (e.g. B*OH*OW % 8 != 0):
        # materialize col for this call — allocates, so only odd shapes
        # (never the steady-state bench models) pay it
        kpad = gw.shape[1]
        col = im2col(x, kh, kw, sh, sw, ph, pw, kpad)
        gemm(dy2, col, ta=True, out=gw, splits=max(splits, 2))
    return gw
