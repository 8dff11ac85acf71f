"""Training driver: composes model step + RCCL all-reduce + fused optimizer,
with optional hipGraph capture of the whole step (launch-bound small models
like the MNIST CNN are exactly the "capture launch-bound inner loops in
hipGraphs" case)."""
from __future__ import annotations

import os
import time
from typing import Callable, Optional, Tuple

import torch

from ..parallel import (all_reduce_grads, get_world_size, is_distributed,
                        oversubscribed)
from ..parallel.ddp import device_step_lock
from .arena import SGD, Adam, Muon
from .layers import SequentialClassifier


def _fn_params(fn):
    import inspect
    try:
        return inspect.signature(fn).parameters
    except (TypeError, ValueError):
        return {}


def _held_tensors(obj, seen=None) -> list:
    """Every tensor that a model's objects hold, layers' buffers included."""
    seen = {} if seen is None else seen
    if id(obj) in seen:
        return []
    if isinstance(obj, torch.Tensor):
        seen[id(obj)] = obj
        return [obj]
    if isinstance(obj, dict):
        inner = list(obj.values())
    elif isinstance(obj, (list, tuple, set)):
        inner = list(obj)
    elif type(obj).__module__.startswith(__name__.split(".")[0]):
        inner = list(getattr(obj, "__dict__", {}).values())
    else:
        return []
    seen[id(obj)] = obj
    return [t for v in inner for t in _held_tensors(v, seen)]


class Trainer:
    def __init__(self, model: SequentialClassifier, optimizer, device="cpu",
                 use_graph: bool = False):
        self.model = model
        self.opt = optimizer
        self.device = torch.device(device)
        # graphs are disabled when ranks time-share one GPU: graph-dispatched
        # kernels corrupt under mid-kernel preemption by the peer process
        # (measured on MI355X, tools/nanverify.py — eager 0/30 bad iterations
        # vs graph 28/30 under identical concurrency); production one-rank-
        # per-GPU runs keep split-graph mode
        self.use_graph = (use_graph and self.device.type == "cuda"
                          and not oversubscribed())
        self._graph = None          # world==1: whole step; world>1: fwd+bwd
        self._graph_opt = None      # world>1: optimizer + mirror refresh
        self._split = False         # world>1 split-graph mode
        # what the graphs write to: layers replace their buffers when another
        # batch size comes by (a prediction, say), and memory that they let go
        # would be other tensors' by the next replay
        self._graph_held = []
        self._static_x = None
        self._static_y = None
        # oversubscribed runs (more ranks than GPUs) serialize device work
        # across ranks: mid-kernel preemption while the peer's kernels/copy
        # tails are in flight corrupts long-running MFMA/LDS wavefront state
        # (measured; see parallel.ddp.device_step_lock). No-op otherwise.
        self._devlock = None

    def _lock(self):
        if self._devlock is None and self.device.type == "cuda" \
                and oversubscribed():
            self._devlock = device_step_lock()
        if self._devlock is None:
            class _Null:
                def __enter__(self): return self
                def __exit__(self, *a): return False
            return _Null()
        return self._devlock

    # full step on given tensors (eager)
    def _step_body(self, x: torch.Tensor, y: torch.Tensor) -> None:
        world = get_world_size()
        gscale = 1.0 / (x.shape[0] * world)
        arena = self.model.arena
        if is_distributed() and oversubscribed():
            # ranks time-share one GPU: serialize compute across ranks and
            # reduce the whole arena once between the locked sections (the
            # lock must not span the collective — the peer needs the device
            # to reach its own all-reduce). Per-layer overlap buys nothing
            # when staging through the host anyway.
            with self._lock():
                self.model.train_step(x, y, gscale=gscale)
            all_reduce_grads(arena.grad)
            with self._lock():
                self.opt.step()
                post = getattr(self.model, "post_opt_step", None)
                if post is not None:
                    post()
            return
        if is_distributed():
            # per-layer async all-reduce overlapped with the backward walk;
            # any params not covered by hooks reduce in one trailing op
            works = []
            covered = []

            def hook(names):
                sl = arena.grad_slice(names)
                if sl is not None and sl.numel():
                    covered.extend(n for n in names if n in arena._offsets)
                    works.append(all_reduce_grads(sl, async_op=True))

            accepts_hook = "grad_hook" in _fn_params(self.model.train_step)
            if accepts_hook:
                self.model.train_step(x, y, gscale=gscale, grad_hook=hook)
            else:
                self.model.train_step(x, y, gscale=gscale)
            leftover = [n for n, _, _ in arena._specs if n not in covered]
            if leftover:
                sl = arena.grad_slice(leftover)
                if sl is not None and sl.numel():
                    works.append(all_reduce_grads(sl, async_op=True))
            for w in works:
                if w is not None:
                    w.wait()
        else:
            self.model.train_step(x, y, gscale=gscale)
        self.opt.step()
        post = getattr(self.model, "post_opt_step", None)
        if post is not None:
            post()

    def step(self, x: torch.Tensor, y: torch.Tensor) -> Tuple[float, float]:
        """One training step. Returns (mean loss, accuracy) — NOTE: these
        device->host reads sync; use step_async inside timed loops."""
        self.step_async(x, y)
        b = x.shape[0]
        return (self.model.loss_sum.item() / b,
                self.model.correct.item() / b)

    def step_async(self, x: torch.Tensor, y: torch.Tensor) -> None:
        if self.use_graph:
            if self._graph is None:
                try:
                    self._capture(x, y)
                except RuntimeError as exc:
                    # capture can fail in environments we cannot pre-test
                    # (e.g. a driver/runtime combination on the 8-GPU node);
                    # a slower eager run beats a crashed scaling bench
                    import sys
                    print(f"[trainer] graph capture failed ({exc}); "
                          "falling back to eager", file=sys.stderr)
                    self.use_graph = False
                    self._graph = None
                    torch.cuda.synchronize()
                    self._step_body(x, y)
                return
            else:
                if self._split:
                    # collectives live OUTSIDE the graphs: one flat SUM
                    # all-reduce of the whole grad arena between the fwd+bwd
                    # graph and the optimizer graph (the
                    # world>1 step must not be launch-bound). Oversubscribed
                    # ranks serialize the replays (lock is a no-op otherwise)
                    with self._lock():
                        self._static_x.copy_(x, non_blocking=True)
                        self._static_y.copy_(y, non_blocking=True)
                        self._graph.replay()
                    all_reduce_grads(self.model.arena.grad)
                    with self._lock():
                        self._graph_opt.replay()
                else:
                    self._static_x.copy_(x, non_blocking=True)
                    self._static_y.copy_(y, non_blocking=True)
                    self._graph.replay()
            return
        self._step_body(x, y)

    def _opt_body(self) -> None:
        self.opt.step()
        post = getattr(self.model, "post_opt_step", None)
        if post is not None:
            post()

    def _capture(self, x: torch.Tensor, y: torch.Tensor) -> None:
        # warm up eagerly (allocates every persistent buffer AND initializes
        # the RCCL communicator before any capture), then capture
        self._split = is_distributed()
        self._static_x = x.clone()
        self._static_y = y.clone()
        world = get_world_size()
        gscale = 1.0 / (x.shape[0] * world)
        if self._split:
            for _ in range(3):
                with self._lock():
                    self.model.train_step(self._static_x, self._static_y,
                                          gscale=gscale)
                all_reduce_grads(self.model.arena.grad)
                with self._lock():
                    self._opt_body()
            torch.cuda.synchronize()
            # thread_local capture: the RCCL/NCCL watchdog thread polls
            # events concurrently; global capture mode would invalidate the
            # capture when it does
            self._graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self._graph,
                                  capture_error_mode="thread_local"):
                self.model.train_step(self._static_x, self._static_y,
                                      gscale=gscale)
            self._graph_opt = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self._graph_opt,
                                  capture_error_mode="thread_local"):
                self._opt_body()
            torch.cuda.synchronize()
            self._graph_held = _held_tensors(self.model)
            return
        for _ in range(3):
            self._step_body(self._static_x, self._static_y)
        torch.cuda.synchronize()
        self._graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self._graph):
            self._step_body(self._static_x, self._static_y)
        torch.cuda.synchronize()
        self._graph_held = _held_tensors(self.model)

    # -- in-training checkpoint/resume (the reference had no
    # epoch-level resume; fit was atomic) --------------------------------
    def save_checkpoint(self, path: str, step: int = 0) -> None:
        state = {"model": self.model.state_dict(), "step": step}
        opt_sd = getattr(self.opt, "state_dict", None)
        if opt_sd is not None:
            state["optimizer"] = opt_sd()
        tmp = path + ".tmp"
        torch.save(state, tmp)
        os.replace(tmp, path)

    def load_checkpoint(self, path: str) -> int:
        state = torch.load(path, map_location="cpu", weights_only=True)
        self.model.load_state_dict(state["model"])
        if "optimizer" in state and hasattr(self.opt, "load_state_dict"):
            self.opt.load_state_dict(state["optimizer"])
        return int(state.get("step", 0))

    def train(self, data_iter, steps: int, log_every: int = 0,
              log_fn: Optional[Callable[[str], None]] = None) -> dict:
        t0 = time.perf_counter()
        samples = 0
        last_loss, last_acc = float("nan"), float("nan")
        for i in range(steps):
            x, y = next(data_iter)
            if log_every and (i + 1) % log_every == 0:
                last_loss, last_acc = self.step(x, y)
                if log_fn:
                    log_fn(f"step {i+1}/{steps} loss={last_loss:.4f} acc={last_acc:.3f}")
            else:
                self.step_async(x, y)
            samples += x.shape[0]
        if self.device.type == "cuda":
            torch.cuda.synchronize()
        dt = time.perf_counter() - t0
        return {"steps": steps, "seconds": dt, "samples": samples,
                "samples_per_sec": samples / dt if dt > 0 else float("inf"),
                "loss": last_loss, "accuracy": last_acc}


def make_sgd(model: SequentialClassifier, lr=0.05, momentum=0.9, wd=0.0) -> SGD:
    return SGD(model.arena, lr=lr, momentum=momentum, weight_decay=wd)


def make_adam(model: SequentialClassifier, lr=1e-3) -> Adam:
    return Adam(model.arena, lr=lr)


def make_muon(model, lr=0.02, momentum=0.95, wd=0.0, exclude=()) -> Muon:
    return Muon(model.arena, lr=lr, momentum=momentum, weight_decay=wd,
                exclude=exclude)
