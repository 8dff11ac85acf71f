"""Explicit-backward NHWC layers over the kernel library.

This is the in-process training engine that replaces the reference's
delegation to TF/keras ``fit`` (SURVEY §3.3 hot loop): a fixed layer graph
with hand-managed forward/backward, all activations in persistent
preallocated buffers (hipGraph-capture friendly — zero allocations in the
steady-state step), parameters/grads in the flat ParamArena.

Gradient-scale convention: the loss head folds 1/(global_batch) into dlogits
(softmax_ce gscale), so every weight grad lands already-averaged and the DDP
all-reduce is a plain SUM.
"""
from __future__ import annotations

import math
import zlib
from typing import List, Optional, Tuple

import torch

from ..ops import functional as F
from .arena import ParamArena


def _pad8(n: int) -> int:
    return (n + 7) // 8 * 8


class Layer:
    def build(self, arena: ParamArena) -> None:  # register params
        pass

    def param_names(self) -> List[str]:
        return []

    def post_opt_step(self) -> None:
        """Refresh derived compute state after an optimizer step (e.g. the
        transposed-weight mirror that keeps dX GEMMs on the fast k-contiguous
        path)."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        raise NotImplementedError

    def backward(self, dy: torch.Tensor) -> Optional[torch.Tensor]:
        raise NotImplementedError


class Conv2dNHWC(Layer):
    """NHWC conv on the fused kernel family (conv_fwd_small / conv_dx /
    conv_dw_c1 / conv1d_* when the shape qualifies — no col/dcol matrices)
    with im2col + MFMA GEMM (+fused bias/ReLU epilogue) as the general
    fallback; 1x1/s1 convs skip im2col entirely."""

    def __init__(self, name: str, in_c: int, out_c: int, kh: int, kw: int,
                 stride: int = 1, pad: int = 0, relu: bool = True,
                 first: bool = False, bias: bool = True,
                 implicit: bool = False, in_used: Optional[int] = None):
        self.name = name
        # input channels that are no padding
        self.in_used = in_c if in_used is None else in_used
        self.bias = bias
        # implicit=True: no col matrix — the fused conv kernels (or the
        # gather-GEMM) handle fwd/dW/dX directly. Measured per model:
        # MNIST + TextCNN default on, ResNet stays on materialized col
        # (3x3 convs are compute-dense; see PERFORMANCE.md A/B entries).
        self.implicit = implicit
        self.in_c, self.out_c = in_c, out_c
        # pad: int (square) or (pad_h, pad_w) — a W==1 sequence conv with
        # h-padding is (p, 0) (padded 1-D convs, r1 fuzz-found gate)
        self.kh, self.kw, self.stride = kh, kw, stride
        self.ph, self.pw = pad if isinstance(pad, (tuple, list)) else (pad, pad)
        self.pad = self.ph  # legacy alias (square users had ph == pw)
        self.relu = relu
        self.first = first  # input layer: skip dX
        self.kdim = kh * kw * in_c
        self.kpad = _pad8(self.kdim)
        # 1x1 stride-1 convs skip im2col entirely (col IS the input)
        self._is_1x1 = (kh == 1 and kw == 1 and stride == 1
                        and self.ph == 0 and self.pw == 0
                        and self.kpad == in_c)
        self.arena: Optional[ParamArena] = None
        self._bufs = {}

    def build(self, arena: ParamArena) -> None:
        self.arena = arena
        std = math.sqrt(2.0 / self.kdim)  # he-init over true fan-in
        kdim, kpad, out_c = self.kdim, self.kpad, self.out_c

        def init_w(shape):
            g = torch.Generator(device="cpu").manual_seed(
                zlib.crc32(self.name.encode()) % (2 ** 31))
            t = torch.zeros(shape, dtype=torch.float32)
            t[:, :kdim] = torch.randn((out_c, kdim), generator=g) * std
            return t

        arena.add(self.name + ".w", (self.out_c, self.kpad), init_w,
                  sides=(out_c, self.kh * self.kw * self.in_used))
        if self.bias:
            arena.add(self.name + ".b", (self.out_c,), torch.zeros(self.out_c))

    def param_names(self) -> List[str]:
        return [self.name + ".w"] + ([self.name + ".b"] if self.bias else [])

    def _alloc(self, B: int, H: int, W: int, dev, dtype):
        OH = (H + 2 * self.ph - self.kh) // self.stride + 1
        OW = (W + 2 * self.pw - self.kw) // self.stride + 1
        key = (B, H, W)
        if self._bufs.get("key") != key:
            M = B * OH * OW
            self._bufs = {
                "key": key, "B": B, "H": H, "W": W, "OH": OH, "OW": OW,
                "y": torch.empty((M, self.out_c), device=dev, dtype=dtype),
            }
            if not self._is_1x1 and not (dev.type == "cuda" and self.implicit):
                # CPU reference path materializes col (GPU gathers it inside
                # the GEMM staging — implicit conv)
                self._bufs["col"] = torch.zeros((M, self.kpad), device=dev, dtype=dtype)
            if not self.first:
                self._bufs["dx"] = torch.empty((B, H, W, self.in_c), device=dev, dtype=dtype)
                if not self._is_1x1 and not (dev.type == "cuda"
                                             and (self._dx_fused_ok(H, W)
                                                  or (self.implicit
                                                      and self._conv1d_ok(W)))):
                    self._bufs["dcol"] = torch.empty((M, self.kpad), device=dev, dtype=dtype)
        return self._bufs

    def _fwd_small_ok(self, H: int, W: int) -> bool:
        # mirror of launch_conv_fwd_small eligibility (x image fits LDS)
        if (self.in_c == 1 and self.kh * self.kw <= 32 and self.kpad >= 32
                and self.out_c <= 64 and self.out_c % 16 == 0
                and (H * W) % 8 == 0 and H * W * 2 + 8192 <= 56 * 1024):
            return True
        return (H * W * (self.in_c * 2 + 16) + 8192 <= 56 * 1024 and
                (self.in_c % 32 == 0 or self.in_c == 16) and
                self.out_c <= 64 and self.out_c % 16 == 0 and
                (self.kh * self.kw * self.in_c) % 32 == 0 and
                (H * W * self.in_c) % 8 == 0)

    def _conv1d_ok(self, W: int) -> bool:
        # mirror of launch_conv1d_* eligibility (W==1 sequence convs).
        # h-padding is fine (the kernels stage zero rows); only w-padding is
        # excluded — w-padding a W==1 input (OW = 2p+1) has no 1-D form, so
        # padded sequence convs use pad=(p, 0) (r1 fuzz-found gate, fixed r2)
        return (W == 1 and self.kw == 1 and self.stride == 1 and
                self.pw == 0 and
                self.in_c % 32 == 0 and self.out_c % 64 == 0 and
                self.out_c <= 128 and (self.kh * self.in_c) % 32 == 0 and
                (64 + self.kh - 1) * (self.in_c * 2 + 16) + 128 + 8192
                <= 56 * 1024 and
                64 * (self.in_c + 4) * 4 + 128 * self.out_c <= 56 * 1024)

    def _dx_fused_ok(self, H: int, W: int) -> bool:
        # mirror of launch_conv_dx eligibility: whole-image dx fits LDS
        hwc = H * W * self.in_c
        return (H * W * (self.in_c + 4) * 4 <= 56 * 1024 and
                (self.in_c % 32 == 0 or self.in_c == 16) and
                hwc % 8 == 0 and self.out_c <= 64 and self.out_c % 8 == 0)

    def _wt(self) -> torch.Tensor:
        # transposed mirror [kpad, out_c] (see Linear._wt)
        if getattr(self, "_wt_buf", None) is None:
            self._wt_buf = self.arena.p(self.name + ".w").t().contiguous()
        return self._wt_buf

    def post_opt_step(self) -> None:
        if getattr(self, "_wt_buf", None) is not None:
            self._wt_buf.copy_(self.arena.p(self.name + ".w").t())

    def forward(self, x: torch.Tensor,
                stats: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``stats``: optional [2, out_c] fp32 workspace — on GPU the GEMM
        epilogue fills per-channel sum/sumsq of the output (the following
        BatchNorm skips its stats pass)."""
        B, H, W, C = x.shape
        assert C == self.in_c
        bufs = self._alloc(B, H, W, x.device, x.dtype)
        self._x = x
        bias = self.arena.pf(self.name + ".b") if self.bias else None
        st = stats if x.is_cuda else None
        if self._is_1x1:
            bufs["col"] = x.view(B * H * W, C)
            F.gemm(bufs["col"], self.arena.p(self.name + ".w"), tb=True,
                   bias=bias, relu=self.relu, out=bufs["y"], stats=st)
        elif x.is_cuda and self.implicit:
            # implicit conv: 1-D tiled kernel (W==1 sequences), small-image
            # fused kernel (x image fits LDS), or im2col gathered inside the
            # GEMM staging as the fallback
            if self._conv1d_ok(W) and F.conv1d_fwd(
                    x, self.arena.p(self.name + ".w"), self.kh, self.ph,
                    bias=bias, relu=self.relu, out=bufs["y"]):
                pass
            elif not (self._fwd_small_ok(H, W) and F.conv2d_fwd_small(
                    x, self.arena.p(self.name + ".w"), self.kh, self.kw,
                    self.stride, self.stride, self.ph, self.pw, bias=bias,
                    relu=self.relu, out=bufs["y"])):
                F.conv2d_fwd_implicit(x, self.arena.p(self.name + ".w"),
                                      self.kh, self.kw, self.stride,
                                      self.stride, self.ph, self.pw,
                                      bias=bias, relu=self.relu,
                                      out=bufs["y"])
            st = None
        else:
            F.im2col(x, self.kh, self.kw, self.stride, self.stride, self.ph,
                     self.pw, self.kpad, out=bufs["col"])
            F.gemm(bufs["col"], self.arena.p(self.name + ".w"), tb=True,
                   bias=bias, relu=self.relu, out=bufs["y"], stats=st)
        self.stats_filled = st is not None
        return bufs["y"].view(B, bufs["OH"], bufs["OW"], self.out_c)

    # True when the following pool's backward already applied our ReLU mask
    relu_bwd_upstream = False

    def backward(self, dy: torch.Tensor,
                 dx_out: Optional[torch.Tensor] = None,
                 dx_accumulate: bool = False,
                 dx_addend: Optional[torch.Tensor] = None,
                 bias_grad_src: Optional[torch.Tensor] = None
                 ) -> Optional[torch.Tensor]:
        """``dx_out``/``dx_accumulate``: on the fused 1-D dX path, write (or
        add) the input grad straight into the caller's buffer — fuses the
        multi-branch grad sum (TextCNN).  Callers must check the returned
        tensor: on fallback paths it is the layer's own dx buffer.

        ``bias_grad_src``: either a small [rows, out_c] matrix or a
        (matrix, u8-mask) pair whose (masked) column sums EQUAL colsum(dy)
        — e.g. the pool-level grad with the ReLU-sentinel idx mask when a
        max pool follows this conv (the pool scatters each value at most
        once, so the sums agree); the bias grad then reads the pool-level
        tensor instead of re-streaming the full dy."""
        bufs = self._bufs
        M = bufs["y"].shape[0]
        dy2 = dy.reshape(M, self.out_c)
        if self.relu and not self.relu_bwd_upstream:
            F.relu_bwd(dy2, bufs["y"], out=dy2)
        # weight grad: dW[outC, kpad] = dY^T @ col, split-K when M is deep
        gw = self.arena.g(self.name + ".w")
        splits = _splitk_heuristic(self.out_c, self.kpad, M)
        if dy2.is_cuda and self.implicit and not self._is_1x1:
            done = (self.in_c == 1 and self.out_c <= 32 and F.conv2d_dw_c1(
                dy2, self._x, gw, self.kh, self.kw, self.stride,
                self.stride, self.ph, self.pw))
            if not done:
                done = F.conv2d_dw_small(dy2, self._x, gw, self.kh, self.kw,
                                         self.stride, self.stride, self.ph,
                                         self.pw)
            if not done:
                F.conv2d_dw_implicit(dy2, self._x, gw, self.kh, self.kw,
                                     self.stride, self.stride, self.ph,
                                     self.pw, splits)
        else:
            F.gemm(dy2, bufs["col"], ta=True, out=gw, splits=splits)
        if self.bias:
            if isinstance(bias_grad_src, tuple):
                F.colsum(bias_grad_src[0], mask=bias_grad_src[1],
                         out=self.arena.g(self.name + ".b"))
            elif bias_grad_src is not None:
                F.colsum(bias_grad_src, out=self.arena.g(self.name + ".b"))
            else:
                F.colsum(dy2, out=self.arena.g(self.name + ".b"))
        if self.first:
            return None
        if self._is_1x1:
            # 1x1/s1 conv: col IS x, so dcol IS dx; dx_addend fuses the
            # residual-join add into the GEMM epilogue (all gemm paths --
            # native, library fallback, CPU reference -- apply it)
            dx = bufs["dx"]
            F.gemm(dy2, self._wt(), tb=True, out=dx.view(M, self.in_c),
                   addend=dx_addend.view(M, self.in_c)
                   if dx_addend is not None else None)
            return dx
        assert dx_addend is None or self._is_1x1, "dx_addend: 1x1 only"
        if dy2.is_cuda and self.implicit and self._conv1d_ok(bufs["W"]):
            tgt = dx_out if dx_out is not None else bufs["dx"]
            if F.conv1d_dx(dy2, self._wt(), self.kh, self.ph, out=tgt,
                           accumulate=dx_accumulate):
                return tgt
        if dy2.is_cuda and self._dx_fused_ok(bufs["H"], bufs["W"]) \
                and F.conv2d_dx_fused(
                dy2, self._wt(), bufs["B"], bufs["H"], bufs["W"], self.in_c,
                self.kh, self.kw, self.stride, self.stride, self.ph,
                self.pw, out=bufs["dx"]):
            return bufs["dx"]
        F.gemm(dy2, self._wt(), tb=True, out=bufs["dcol"])
        F.col2im(bufs["dcol"], bufs["B"], bufs["H"], bufs["W"], self.in_c,
                 self.kh, self.kw, self.stride, self.stride, self.ph,
                 self.pw, out=bufs["dx"])
        return bufs["dx"]


class MaxPool2dNHWC(Layer):
    def __init__(self, k: int = 2, stride: Optional[int] = None,
                 kw: Optional[int] = None, sw: Optional[int] = None,
                 pad: int = 0):
        self.kh = k
        self.kw = kw if kw is not None else k
        self.sh = stride or k
        self.sw = sw if sw is not None else (stride or self.kw)
        self.ph = self.pw = pad
        self._bufs = {}

    # aliases used by models that retune pooling per sequence length
    def set_window(self, kh: int, kw: int, sh: Optional[int] = None,
                   sw: Optional[int] = None) -> None:
        self.kh, self.kw = kh, kw
        self.sh = sh if sh is not None else kh
        self.sw = sw if sw is not None else kw

    # set by SequentialClassifier when the preceding layer is a ReLU conv:
    # the conv's ReLU backward mask folds into this kernel (relu_y = the
    # pool input) and the conv skips its own relu_bwd pass.
    fuse_relu = False

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        self._bufs["shape"] = x.shape
        # fuse_relu: the upstream conv's ReLU bwd folds into the argmax idx
        # (sentinel 255 where max <= 0), so backward needs no relu_y stream
        out, idx = F.maxpool2d(x, self.kh, self.kw, self.sh, self.sw,
                               self.ph, self.pw, relu_mask=self.fuse_relu)
        self._bufs["idx"] = idx
        if "dx" not in self._bufs or self._bufs["dx"].shape != x.shape:
            self._bufs["dx"] = torch.empty_like(x)
        return out

    def backward(self, dy: torch.Tensor) -> torch.Tensor:
        B, H, W, C = self._bufs["shape"]
        self._last_dy = dy                    # pool-level grad (bias source)
        return F.maxpool2d_bwd(dy, self._bufs["idx"], H, W, self.kh, self.kw,
                               self.sh, self.sw, self.ph, self.pw,
                               out=self._bufs["dx"], relu_y=None)


class Flatten(Layer):
    def forward(self, x: torch.Tensor) -> torch.Tensor:
        self._shape = x.shape
        return x.reshape(x.shape[0], -1)

    def backward(self, dy: torch.Tensor) -> torch.Tensor:
        return dy.reshape(self._shape)


class Linear(Layer):
    def __init__(self, name: str, in_f: int, out_f: int, relu: bool = False,
                 in_used: Optional[int] = None, out_used: Optional[int] = None):
        self.name = name
        # features and outputs that are no padding
        self.in_used, self.out_used = in_used, out_used
        self.in_f, self.out_f = in_f, out_f
        self.relu = relu
        self.arena: Optional[ParamArena] = None
        self._bufs = {}

    def build(self, arena: ParamArena) -> None:
        self.arena = arena
        std = math.sqrt(2.0 / self.in_f)
        g = torch.Generator(device="cpu").manual_seed(zlib.crc32(self.name.encode()) % (2 ** 31))
        arena.add(self.name + ".w", (self.out_f, self.in_f),
                  torch.randn((self.out_f, self.in_f), generator=g) * std,
                  sides=(self.out_used or self.out_f, self.in_used or self.in_f))
        arena.add(self.name + ".b", (self.out_f,), torch.zeros(self.out_f))

    def param_names(self) -> List[str]:
        return [self.name + ".w", self.name + ".b"]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        M = x.shape[0]
        if self._bufs.get("M") != M:
            self._bufs = {"M": M,
                          "y": torch.empty((M, self.out_f), device=x.device, dtype=x.dtype),
                          "dx": torch.empty((M, self.in_f), device=x.device, dtype=x.dtype)}
        self._bufs["x"] = x
        F.gemm(x, self.arena.p(self.name + ".w"), tb=True,
               bias=self.arena.pf(self.name + ".b"), relu=self.relu,
               out=self._bufs["y"])
        return self._bufs["y"]

    def _wt(self) -> torch.Tensor:
        # transposed mirror [in_f, out_f]: dX = dY @ W runs as the fast (F,T)
        # GEMM (k-contiguous B) instead of the transpose-staged (F,F) path
        if getattr(self, "_wt_buf", None) is None:
            self._wt_buf = self.arena.p(self.name + ".w").t().contiguous()
        return self._wt_buf

    def post_opt_step(self) -> None:
        if getattr(self, "_wt_buf", None) is not None:
            self._wt_buf.copy_(self.arena.p(self.name + ".w").t())

    def backward(self, dy: torch.Tensor) -> torch.Tensor:
        bufs = self._bufs
        if self.relu:
            F.relu_bwd(dy, bufs["y"], out=dy)
        gw = self.arena.g(self.name + ".w")
        splits = _splitk_heuristic(self.out_f, self.in_f, bufs["M"])
        F.gemm(dy, bufs["x"], ta=True, out=gw, splits=splits)
        F.colsum(dy, out=self.arena.g(self.name + ".b"))
        F.gemm(dy, self._wt(), tb=True, out=bufs["dx"])
        return bufs["dx"]


def _splitk_heuristic(m: int, n: int, k: int) -> int:
    """Split-K factor for the dW GEMM C[m,n] with reduction depth k: fill the
    256-CU chip (~512 blocks of 32x64 tiles) without shredding k."""
    bm = 64 if m >= 64 else 32   # mirror the split-K tile selection
    base_blocks = ((m + bm - 1) // bm) * ((n + 63) // 64)
    if base_blocks >= 2048 or k < 2048:
        return 1
    return max(1, min(2048 // base_blocks, k // 1024))


class SequentialClassifier:
    """A fixed feed-forward classifier on the explicit-backward engine, with
    the padded-class softmax-CE head (padded logits masked in the kernel)."""

    def __init__(self, layers: List[Layer], num_classes: int, device="cpu",
                 seed: int = 0):
        self.layers = layers
        self.num_classes = num_classes
        # fuse conv-ReLU backward into the following maxpool's backward
        for prev, nxt in zip(layers, layers[1:]):
            if (isinstance(prev, Conv2dNHWC) and prev.relu
                    and isinstance(nxt, MaxPool2dNHWC)):
                nxt.fuse_relu = True
                prev.relu_bwd_upstream = True
                prev._fused_pool = nxt  # bias grad from the pool-level grad
        head = layers[-1] if layers else None
        if isinstance(head, Linear) and head.out_used is None:
            head.out_used = min(num_classes, head.out_f)
        self.arena = ParamArena(device)
        for lay in layers:
            lay.build(self.arena)
        self.arena.finalize(seed)
        dev = torch.device(device)
        self.loss_sum = torch.zeros(1, dtype=torch.float32, device=dev)
        self.correct = torch.zeros(1, dtype=torch.int32, device=dev)
        self._dlogits = None

    @property
    def cpad(self) -> int:
        # classifier head output width (padded to 8/16 for aligned GEMMs)
        return self.layers[-1].out_f

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        for lay in self.layers:
            x = lay.forward(x)
        return x

    def train_step(self, x: torch.Tensor, y: torch.Tensor,
                   gscale: Optional[float] = None,
                   grad_hook=None) -> Tuple[torch.Tensor, torch.Tensor]:
        """One fused fwd+bwd. Returns (loss_sum, correct) device tensors;
        optimizer step is separate (Trainer composes allreduce between).
        ``grad_hook(param_names)`` fires after each layer's grads are final
        (the DDP overlap point)."""
        if gscale is None:
            gscale = 1.0 / x.shape[0]
        logits = self.forward(x)
        if self._dlogits is None or self._dlogits.shape != logits.shape:
            self._dlogits = torch.empty_like(logits)
        self.loss_sum.zero_()
        self.correct.zero_()
        F.softmax_ce(logits, y, self._dlogits, self.loss_sum, self.correct,
                     cvalid=self.num_classes, gscale=gscale)
        dy = self._dlogits
        for lay in reversed(self.layers):
            if (isinstance(lay, Conv2dNHWC)
                    and getattr(lay, "_fused_pool", None) is not None
                    and lay.bias and dy is not None):
                # colsum(dconv) == colsum(pool-level dy masked by the
                # ReLU-sentinel idx): sum the SMALL tensor (the non-overlap
                # pool scatters each value at most once)
                pool = lay._fused_pool
                pdy, pidx = pool._last_dy, pool._bufs["idx"]
                dy = lay.backward(dy, bias_grad_src=(
                    pdy.reshape(-1, lay.out_c),
                    pidx.reshape(-1, lay.out_c)))
            else:
                dy = lay.backward(dy)
            if grad_hook and lay.param_names():
                grad_hook(lay.param_names())
            if dy is None:
                break
        return self.loss_sum, self.correct

    def post_opt_step(self) -> None:
        for lay in self.layers:
            lay.post_opt_step()

    @torch.no_grad()
    def predict(self, x: torch.Tensor) -> torch.Tensor:
        logits = self.forward(x)
        return F.argmax_rows(logits, self.num_classes)

    # -- checkpoint/resume ------------------------------------
    def state_dict(self):
        return self.arena.state_dict()

    def load_state_dict(self, sd):
        self.arena.load_state_dict(sd)
        self.post_opt_step()  # refresh transposed weight mirrors


class Embedding(Layer):
    """Token embedding gather; backward scatter-adds into the grad arena
    (embedding.hip; fp32 atomics)."""

    def __init__(self, name: str, vocab: int, dim: int):
        assert dim % 8 == 0, "embedding dim must be 8-aligned"
        self.name = name
        self.vocab, self.dim = vocab, dim
        self.arena: Optional[ParamArena] = None
        self._ids = None
        self._out = None

    def build(self, arena: ParamArena) -> None:
        self.arena = arena
        g = torch.Generator(device="cpu").manual_seed(
            zlib.crc32(self.name.encode()) % (2 ** 31))
        arena.add(self.name + ".w", (self.vocab, self.dim),
                  torch.randn((self.vocab, self.dim), generator=g) * 0.05)

    def param_names(self):
        return [self.name + ".w"]

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        from ..ops import functional as F_
        self._ids = ids
        if self._out is None or self._out.shape[:ids.dim()] != ids.shape:
            self._out = torch.empty(*ids.shape, self.dim,
                                    device=self.arena.mirror.device,
                                    dtype=torch.bfloat16)
        F_.embedding(ids, self.arena.p(self.name + ".w"), out=self._out)
        return self._out

    def backward(self, dy: torch.Tensor) -> None:
        from ..ops import functional as F_
        g = self.arena.g(self.name + ".w")
        g.zero_()  # scatter-add accumulates; arena grads are per-step
        F_.embedding_bwd(self._ids, dy, g)
        return None


class BatchNormReLU(Layer):
    '''Per-channel BN (+fused ReLU) over NHWC activations (batchnorm.hip).
    Running stats live on the layer (non-trainable state, included in the
    model's extra-state checkpoint); gamma/beta in the arena.'''

    def __init__(self, name: str, channels: int, relu: bool = True,
                 eps: float = 1e-5, momentum: float = 0.1):
        assert channels % 8 == 0
        self.name = name
        self.c = channels
        self.relu = relu
        self.residual_relu = True   # fused-join z = relu(bn(x) + residual)
        self.eps = eps
        self.momentum = momentum
        self.training = True
        self.arena: Optional[ParamArena] = None
        self._bufs = {}

    def build(self, arena: ParamArena) -> None:
        self.arena = arena
        arena.add(self.name + ".g", (self.c,), torch.ones(self.c))
        arena.add(self.name + ".b", (self.c,), torch.zeros(self.c))
        # running stats are keyed only on C and live for the model's lifetime
        # (NOT in the shape-keyed _bufs dict: a batch-size change must not
        # reset them, and load_extra_state must work before any forward)
        self.running_mean = torch.zeros(self.c, device=arena.device)
        self.running_var = torch.ones(self.c, device=arena.device)

    def param_names(self):
        return [self.name + ".g", self.name + ".b"]

    def scratch(self, dev) -> torch.Tensor:
        """[2, C] sum/sumsq workspace — exposed so the producing conv's GEMM
        epilogue can fill it (fused bn_stats)."""
        if getattr(self, "_scratch", None) is None:
            self._scratch = torch.zeros((2, self.c), device=dev)
        return self._scratch

    def _alloc(self, shape, dev):
        if self._bufs.get("shape") != shape:
            M = 1
            for d in shape[:-1]:
                M *= d
            self._bufs = {
                "shape": shape, "M": M,
                "y": torch.empty((M, self.c), device=dev, dtype=torch.bfloat16),
                "dx": torch.empty((M, self.c), device=dev, dtype=torch.bfloat16),
                "mean": torch.zeros(self.c, device=dev),
                "invstd": torch.ones(self.c, device=dev),
                "scratch": self.scratch(dev),
            }
        return self._bufs

    def forward(self, x: torch.Tensor, stats_ready: bool = False,
                residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``residual``: fused join z = relu(bn(x) + residual) — the ResNet
        bottleneck add without a separate add_relu pass. The residual only
        changes the forward output; bn backward w.r.t. x is unaffected
        (callers mask dz by z themselves, as with add_relu)."""
        bufs = self._alloc(tuple(x.shape), x.device)
        x2 = x.reshape(bufs["M"], self.c)
        self._x2 = x2
        relu = self.relu or (residual is not None and self.residual_relu)
        gamma = self.arena.pf(self.name + ".g")
        beta = self.arena.pf(self.name + ".b")
        if self.training:
            run = ((self.running_mean, self.running_var) if x.is_cuda
                   else None)
            F.bn_fwd_train(x2, gamma, beta, self.eps, bufs["y"], bufs["mean"],
                           bufs["invstd"], bufs["scratch"], relu,
                           stats_ready=stats_ready and x.is_cuda,
                           residual=residual, running=run,
                           momentum=self.momentum)
            if not x.is_cuda:
                m = self.momentum
                self.running_mean.mul_(1 - m).add_(bufs["mean"], alpha=m)
                var = bufs["invstd"].square().reciprocal() - self.eps
                self.running_var.mul_(1 - m).add_(var, alpha=m)
        else:
            F.bn_fwd_eval(x2, gamma, beta, self.running_mean,
                          self.running_var, self.eps, bufs["y"], relu,
                          residual=residual)
        return bufs["y"].view(x.shape)

    def backward(self, dy: torch.Tensor) -> torch.Tensor:
        bufs = self._bufs
        dy2 = dy.reshape(bufs["M"], self.c)
        F.bn_bwd(dy2, bufs["y"], self._x2, bufs["mean"], bufs["invstd"],
                 self.arena.pf(self.name + ".g"),
                 self.arena.g(self.name + ".g"), self.arena.g(self.name + ".b"),
                 bufs["dx"], self.relu)
        return bufs["dx"].view(dy.shape)

    # checkpointable non-arena state
    def extra_state(self):
        return {self.name + ".running_mean": self.running_mean.cpu(),
                self.name + ".running_var": self.running_var.cpu()}

    def load_extra_state(self, sd):
        if self.name + ".running_mean" in sd:
            self.running_mean.copy_(sd[self.name + ".running_mean"].to(
                self.running_mean.device))
            self.running_var.copy_(sd[self.name + ".running_var"].to(
                self.running_var.device))


class LayerNorm(Layer):
    '''Layer norm over the last axis (layernorm.hip), the norm that does not
    depend on the batch: same result for one text as inside a batch, no
    running state. gamma/beta in the arena.'''

    def __init__(self, name: str, channels: int, eps: float = 1e-5):
        assert 1 <= channels <= 32768
        self.name = name
        self.c = channels
        self.eps = eps
        self.arena: Optional[ParamArena] = None
        self._bufs = {}

    def build(self, arena: ParamArena) -> None:
        self.arena = arena
        arena.add(self.name + ".g", (self.c,), torch.ones(self.c))
        arena.add(self.name + ".b", (self.c,), torch.zeros(self.c))

    def param_names(self):
        return [self.name + ".g", self.name + ".b"]

    def _alloc(self, x):
        key = (tuple(x.shape), x.dtype)
        if self._bufs.get("key") != key:
            M = x.numel() // self.c
            dev = x.device
            self._bufs = {
                "key": key, "M": M,
                "y": torch.empty((M, self.c), device=dev, dtype=x.dtype),
                "dx": torch.empty((M, self.c), device=dev, dtype=x.dtype),
                "mean": torch.empty(M, device=dev),
                "invstd": torch.empty(M, device=dev),
            }
        return self._bufs

    def _rows(self, t: torch.Tensor) -> torch.Tensor:
        # any view: the kernels take any row stride, but whole rows
        t = t.reshape(self._bufs["M"], self.c)
        return t if t.stride(1) == 1 or self.c == 1 else t.contiguous()

    def forward(self, x: torch.Tensor,
                residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``residual``: normalise x + residual; the sum stays in
        ``self.sum`` (x's shape) for the skip path."""
        assert x.shape[-1] == self.c
        bufs = self._alloc(x)
        x2 = self._rows(x)
        self._x2 = x2
        if residual is not None:
            if "sum" not in bufs:
                bufs["sum"] = torch.empty_like(bufs["y"])
            self._x2 = bufs["sum"]
            residual = self._rows(residual)
        F.layernorm_fwd(x2, self.arena.pf(self.name + ".g"),
                        self.arena.pf(self.name + ".b"), self.eps, bufs["y"],
                        mean=bufs["mean"], invstd=bufs["invstd"],
                        residual=residual,
                        sum_out=bufs["sum"] if residual is not None else None)
        self.sum = self._x2.view(x.shape) if residual is not None else None
        return bufs["y"].view(x.shape)

    def backward(self, dy: torch.Tensor,
                 dskip: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``dskip``: gradient that reached ``self.sum`` past the norm. The
        result is the gradient of x and of the residual alike."""
        bufs = self._bufs
        if dskip is not None:
            dskip = self._rows(dskip)
        F.layernorm_bwd(self._rows(dy), self._x2, bufs["mean"],
                        bufs["invstd"], self.arena.pf(self.name + ".g"),
                        self.arena.g(self.name + ".g"),
                        self.arena.g(self.name + ".b"), bufs["dx"],
                        dskip=dskip)
        return bufs["dx"].view(dy.shape)


class AvgPoolGlobal(Layer):
    '''Global average pool [B,H,W,C] -> [B,C] (batchnorm.hip kernels).'''

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        self._shape = x.shape
        B, H, W, C = x.shape
        if not hasattr(self, "_out") or self._out.shape[0] != B:
            self._out = torch.empty((B, C), device=x.device, dtype=x.dtype)
            self._dx = torch.empty_like(x)
        return F.avgpool_global(x, out=self._out)

    def backward(self, dy: torch.Tensor) -> torch.Tensor:
        B, H, W, C = self._shape
        return F.avgpool_global_bwd(dy, H, W, out=self._dx)
