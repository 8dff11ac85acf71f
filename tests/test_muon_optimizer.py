"""The Muon optimizer and layer norm inside the engine: parameter split, steps
against the operators they are made of, checkpoints, captured steps, and a
small network's gradients."""
import copy
import io
import os

import pytest
import torch
import torch.multiprocessing as mp

from learningorchestra_amd.data.synthetic import imdb_batch
from learningorchestra_amd.engine.arena import Muon, ParamArena
from learningorchestra_amd.engine.layers import (Conv2dNHWC, Flatten,
                                                 LayerNorm, Linear,
                                                 MaxPool2dNHWC,
                                                 SequentialClassifier)
from learningorchestra_amd.engine.trainer import (Trainer, _held_tensors,
                                                  make_muon)
from learningorchestra_amd.models.mnist_cnn import build_mnist_cnn
from learningorchestra_amd.models.resnet import ResNet
from learningorchestra_amd.models.tabular import MLPClassifier
from learningorchestra_amd.models.textcnn import build_textcnn
from learningorchestra_amd.models.zoo import TextCNNClassifier
from learningorchestra_amd.ops import functional as F

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _arena(device):
    a = ParamArena(device)
    a.add("emb.w", (30, 8), 0.1)
    a.add("conv.w", (16, 40), 0.1)
    a.add("conv.b", (16,), 0.1)
    a.add("ln.g", (24,), 0.1)
    a.add("row.w", (1, 24), 0.1)
    a.add("tall.w", (70, 9), 0.1)
    a.add("head.w", (8, 70), 0.1)
    a.finalize(seed=3)
    return a


def _grads(arena, seed):
    g = torch.randn(arena.numel, generator=torch.Generator().manual_seed(seed))
    arena.grad.copy_(g * 1e-2)
    for name, _, _ in arena._specs:   # the padding holds no gradient
        off, n = arena._offsets[name]
        arena.grad[off + n:off + (n + 7) // 8 * 8] = 0


@pytest.mark.parametrize("device", DEVICES)
def test_matrices_and_the_rest(device):
    a = _arena(device)
    opt = Muon(a, exclude=("emb.w", "head.w"))
    assert opt.matrices == ["conv.w", "tall.w"]
    assert Muon(_arena(device)).matrices == ["emb.w", "conv.w", "tall.w",
                                             "head.w"]
    with pytest.raises(ValueError):
        Muon(a, exclude=("nothing",))
    with pytest.raises(ValueError):
        Muon(a, exclude=("emb.w", "conv.w", "tall.w", "head.w"))


@pytest.mark.parametrize("device", DEVICES)
def test_step_is_its_operators(device):
    a, b = _arena(device), _arena(device)
    opt = Muon(a, lr=0.03, momentum=0.9, weight_decay=0.1, exclude=("emb.w",),
               adam_lr=0.01)
    views = [(b._offsets[n][0], *b.p(n).shape) for n in opt.matrices]
    plan = F.MuonPlan(views, b.numel, device)
    mom, m2 = torch.zeros_like(b.master), torch.zeros_like(b.master)
    t = torch.zeros(1, dtype=torch.int32, device=device)
    for seed in range(3):
        for arena in (a, b):
            _grads(arena, seed)
        opt.step(gscale=0.5)
        t += 1
        F.muon_step(plan, b.master, b.grad, mom, b.mirror, 0.03, 0.9, 0.1, 0.5)
        for name, shape, _ in b._specs:
            if name in opt.matrices:
                continue
            off, n = b._offsets[name]
            sl = slice(off, off + (n + 7) // 8 * 8)
            F.adam_step(b.master[sl], b.grad[sl], mom[sl], m2[sl],
                        b.mirror[sl], 0.01, 0.9, 0.999, 1e-8, 0.1, t, 0.5)
        for x, y in ((a.master, b.master), (a.mirror, b.mirror),
                     (opt.mom, mom), (opt.m2, m2)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("device", DEVICES)
def test_checkpoint(device):
    a = _arena(device)
    opt = Muon(a, lr=0.03, exclude=("emb.w",))
    for seed in range(2):
        _grads(a, seed)
        opt.step()
    buf = io.BytesIO()
    torch.save({"model": a.state_dict(), "optimizer": opt.state_dict()}, buf)
    buf.seek(0)
    b = _arena(device)
    again = Muon(b, exclude=("emb.w",))
    saved = torch.load(buf, map_location="cpu", weights_only=True)
    b.load_state_dict(saved["model"])
    again.load_state_dict(saved["optimizer"])
    for seed in range(2, 4):
        for arena, o in ((a, opt), (b, again)):
            _grads(arena, seed)
            o.step()
    assert torch.equal(a.master, b.master)


@pytest.mark.gpu
def test_captured_steps():
    """A captured step goes on as eager ones do, Adam's count included."""
    a, b = _arena("cuda"), _arena("cuda")
    eager, captured = (Muon(x, exclude=("emb.w",)) for x in (a, b))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step()
    for seed in range(4):
        _grads(a, seed)
        _grads(b, seed)
        eager.step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a.master, b.master)
        assert torch.equal(a.mirror, b.mirror)
    assert int(captured.t) == 4


@pytest.mark.gpu
def test_ranges_beyond_32_bits():
    gen = torch.Generator().manual_seed(4)
    near = [torch.rand(64, generator=gen).cuda() for _ in range(4)]
    near.append(near[0].bfloat16())
    far = [torch.empty(2 ** 31 + 64, dtype=t.dtype, device="cuda") for t in near]
    for f, t in zip(far, near):
        f[2 ** 31:] = t
    step = torch.ones(1, dtype=torch.int32, device="cuda")
    for at, arena in ((0, near), (2 ** 31, far)):
        r = F.AdamRanges([(at + 8, at + 24), (at + 40, at + 64)], at + 64, "cuda")
        F.adam_ranges(r, *arena, 0.1, 0.9, 0.99, 1e-8, 0.01, step)
    for f, t in zip(far, near):
        assert torch.equal(f[2 ** 31:], t)


def test_ranges_do_not_overlap():
    for bad in ([(0, 16), (8, 24)], [(8, 24), (0, 16)], [(0, 8), (0, 8)]):
        with pytest.raises(ValueError):
            F.AdamRanges(bad, 64, "cpu")
    F.AdamRanges([(8, 24), (0, 8)], 64, "cpu")


@pytest.mark.parametrize("device", DEVICES)
def test_ranges_refusals(device):
    for bad in ([(0, 12)], [(4, 16)], [(16, 8)], [(0, 72)], [(-8, 8)]):
        with pytest.raises(ValueError):
            F.AdamRanges(bad, 64, device)
    r = F.AdamRanges([(8, 16)], 64, device)
    z = torch.zeros(72, device=device)
    with pytest.raises(RuntimeError):
        F.adam_ranges(r, z, z, z, z, z.bfloat16(), 0.1, 0.9, 0.99, 1e-8, 0.0, 1)
    # no ranges: nothing moves
    w = torch.ones(64, device=device)
    F.adam_ranges(F.AdamRanges([], 64, device), w, w.clone(), w.clone(),
                  w.clone(), w.bfloat16(), 0.1, 0.9, 0.99, 1e-8, 0.0, 1)
    assert bool((w == 1).all())


def _network(device):
    return SequentialClassifier(
        [LayerNorm("ln0", 48), Linear("fc1", 48, 64, relu=True),
         LayerNorm("ln1", 64), Linear("fc2", 64, 16)], num_classes=10,
        device=device)


@pytest.mark.parametrize("device", DEVICES)
def test_network_gradients_and_steps(device):
    """Layer norms between linear layers, stepped by Muon. Gradients agree with
    autograd in fp32: about 16 roundings to bf16 of values and gradients lie
    between a parameter and the loss, each off by 2^-8 at most."""
    m = _network(device)
    gen = torch.Generator().manual_seed(5)
    x = (torch.randn(96, 48, generator=gen) * 2 + 1).bfloat16().to(device)
    y = torch.randint(0, 10, (96,), generator=gen).to(device)
    for name in ("ln0", "ln1"):
        m.arena.pf(name + ".g").mul_(1.25)
        m.arena.pf(name + ".b").add_(0.25)
    m.arena.mirror.copy_(m.arena.master)
    m.post_opt_step()
    m.train_step(x, y)
    p = {n: m.arena.pf(n).detach().cpu().clone().requires_grad_()
         for n, _, _ in m.arena._specs}

    def norm(t, name):
        mu = t.mean(1, keepdim=True)
        z = (t - mu) / ((t - mu).square().mean(1, keepdim=True) + 1e-5).sqrt()
        return z * p[name + ".g"] + p[name + ".b"]

    h = norm(x.cpu().float(), "ln0") @ p["fc1.w"].T + p["fc1.b"]
    h = norm(torch.relu(h), "ln1") @ p["fc2.w"].T + p["fc2.b"]
    torch.nn.functional.cross_entropy(h[:, :10], y.cpu()).backward()
    for n, t in p.items():
        got = m.arena.g(n).cpu()
        assert (got - t.grad).norm() <= 16 * 2 ** -8 * t.grad.norm() + 1e-6, n
    trainer = Trainer(m, make_muon(m, exclude=("fc2.w",)), device=device)
    before = m.arena.state_dict()
    for _ in range(3):
        trainer.step_async(x, y)
    after = m.arena.state_dict()
    assert all(bool(torch.isfinite(v).all()) for v in after.values())
    assert all(not torch.equal(before[n], after[n]) for n in p)
    assert torch.equal(m.arena.mirror, m.arena.master.bfloat16())
    assert m.predict(x).shape == (96,)


@pytest.mark.parametrize("device", DEVICES)
def test_textcnn_with_both(device):
    m = build_textcnn(device, vocab=500, emb_dim=32, filters=64,
                      layer_norm=True)
    opt = make_muon(m, exclude=("emb.w", "fc.w"))
    assert opt.matrices == ["conv3.w", "conv4.w", "conv5.w"]
    hooked = []
    ids, y = (t.to(device) for t in imdb_batch(16, seq_len=24, vocab=500,
                                               seed=0))
    m.train_step(ids, y, grad_hook=hooked.extend)
    assert sorted(hooked) == sorted(n for n, _, _ in m.arena._specs)
    assert all(float(m.arena.g(n).abs().sum()) > 0 for n in
               ("ln_emb.g", "ln_emb.b", "ln_cat.g", "ln_cat.b", "emb.w"))
    trainer = Trainer(m, opt, device=device)
    for _ in range(2):
        trainer.step_async(ids, y)
    assert bool(torch.isfinite(m.arena.master).all())
    assert m.predict(ids).shape == (16,)
    # one text's norm is the same alone and in its batch
    feats = torch.randn(16, 192).bfloat16().to(device)
    whole = m.ln_cat.forward(feats).clone()
    assert torch.equal(m.ln_cat.forward(feats[5:6].contiguous()), whole[5:6])


@pytest.mark.parametrize("device", DEVICES)
def test_classifier_options(device):
    with pytest.raises(ValueError):
        TextCNNClassifier(vocab=50, optimizer="other", device=device)
    ids, y = imdb_batch(32, seq_len=16, vocab=50, seed=1)
    c = TextCNNClassifier(vocab=50, emb_dim=32, filters=64, batch_size=16,
                          device=device, layer_norm=True, optimizer="muon",
                          lr=0.02)
    hist = c.fit(ids.numpy(), y.numpy(), epochs=2)
    assert all(v == v for v in hist["loss"])
    assert c.predict(ids.numpy()).shape == (32,)
    d = TextCNNClassifier(device=device, **c.lo_spec)   # as stored and loaded
    d.load_state_dict(c.state_dict())
    assert (d.predict(ids.numpy()) == c.predict(ids.numpy())).all()


def _worker(rank, world, port, q):
    os.environ.update({"RANK": str(rank), "WORLD_SIZE": str(world),
                       "LOCAL_RANK": str(rank),
                       "MASTER_ADDR": "127.0.0.1", "MASTER_PORT": str(port)})
    import torch.distributed as dist
    from learningorchestra_amd.parallel import init_distributed
    try:
        torch.set_num_threads(1)
        init_distributed(backend="gloo")
        m = _network("cpu")
        trainer = Trainer(m, make_muon(m, exclude=("fc2.w",)), device="cpu")
        gen = torch.Generator().manual_seed(50 + rank)
        x = torch.randn(32, 48, generator=gen).bfloat16()
        y = torch.randint(0, 10, (32,), generator=gen)
        for _ in range(3):
            trainer.step_async(x, y)
        q.put((rank, m.arena.master.tolist()))
        dist.destroy_process_group()
    except Exception as exc:  # pragma: no cover
        q.put((rank, f"ERROR: {exc!r}"))


@pytest.mark.timeout(240)
def test_two_ranks_stay_identical():
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, 2, 29547, q))
             for r in range(2)]
    for p in procs:
        p.start()
    results = [q.get(timeout=220)[1] for _ in range(2)]
    for p in procs:
        p.join(timeout=30)
    assert not isinstance(results[0], str), results[0]
    assert results[0] == results[1]


def _orthogonal64(u):
    x = u / (u.norm() + 1e-7)
    a, b, c = F.NS_COEFFS
    for _ in range(5):
        s = x @ x.T
        x = a * x + (b * s + c * (s @ s)) @ x
    return x


@pytest.mark.parametrize("device", DEVICES)
def test_padding_does_not_shorten_the_steps(device):
    """Weights stored with rows or columns of padding (a convolution's taps,
    the head's classes, the stem's channels) move as their own sides say. The
    tolerance is that of fp32 steps, 1800 sqrt(K) 2^-24 of the step: three sums
    of K products a step, grown by |p'| < 4 in each later one. The padded sides
    would make it up to 28 % shorter."""
    m = SequentialClassifier(
        [Conv2dNHWC("wide", 1, 32, 5, 5, first=True), MaxPool2dNHWC(2),
         Flatten(), Linear("narrow", 4 * 4 * 32, 8), Linear("fc", 8, 16)],
        num_classes=10, device=device)
    assert m.arena.p("wide.w").shape == (32, 32)
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(40, 12, 12, 1, generator=gen).bfloat16().to(device)
    y = torch.randint(0, 10, (40,), generator=gen).to(device)
    m.train_step(x, y)
    opt = make_muon(m, lr=0.1, momentum=0.5)
    own = {"wide.w": (32, 25), "narrow.w": (8, 512), "fc.w": (10, 8)}
    assert opt.matrices == list(own)
    before = {n: m.arena.pf(n).double().cpu() for n in own}
    opt.step()
    for n, (rows, cols) in own.items():
        g = m.arena.g(n).double().cpu()
        assert bool((g[rows:] == 0).all()) and bool((g[:, cols:] == 0).all())
        o = _orthogonal64(1.5 * g)
        step = 0.1 * max(1.0, rows / cols) ** 0.5 * o
        err = m.arena.pf(n).double().cpu() - (before[n] - step)
        tol = 1800 * max(g.shape) ** 0.5 * 2 ** -24 * step.norm() \
            + 4 * 2 ** -24 * (before[n].norm() + step.norm())
        assert err.norm() <= tol, n


def test_models_know_their_padding():
    assert build_mnist_cnn().arena.sides == {"conv1.w": (32, 25),
                                             "fc2.w": (10, 256)}
    assert build_textcnn("cpu", vocab=50).arena.sides == {"fc.w": (2, 384)}
    r = ResNet((1, 1, 1, 1), num_classes=10, width=16).arena.sides
    assert r == {"stem.w": (16, 147), "fc.w": (10, 512)}
    c = MLPClassifier(hidden=(16,), epochs=1, device="cpu")
    c.fit(torch.randn(20, 5).numpy(), [0, 1] * 10)
    assert c.model.arena.sides == {"mlp.l0.w": (16, 5), "mlp.head.w": (2, 16)}


@pytest.mark.parametrize("device", DEVICES)
def test_sides_of_a_plan(device):
    """In any order of the views, and refused where they are no part of them."""
    views = [(64, 8, 4), (0, 6, 4)]
    a = F.MuonPlan(views, 96, device, sides=[(8, 2), (6, 1)])
    assert a.gains == [2.0, 6 ** 0.5]
    b = F.MuonPlan(views[::-1], 96, device, sides=[(6, 1), (8, 2)])
    none = F.MuonPlan(views, 96, device)
    g = torch.zeros(96)
    gen = torch.Generator().manual_seed(8)
    g[0:24].view(6, 4)[:, :1] = torch.randn(6, 1, generator=gen)
    g[64:96].view(8, 4)[:, :2] = torch.randn(8, 2, generator=gen)
    got = []
    for plan in (a, b, none, copy.deepcopy(a)):
        w, m = (torch.zeros(96, device=device) for _ in range(2))
        F.muon_step(plan, w, g.to(device), m, w.bfloat16(), lr=0.5)
        got.append(w.cpu())
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[3])
    for sl, ratio in ((slice(0, 24), 4 ** 0.5), (slice(64, 96), 2 ** 0.5)):
        # two roundings apart: of the factors, and of the products
        assert ((got[0] - ratio * got[2])[sl].abs()
                <= 4 * 2 ** -24 * got[0][sl].abs()).all()
        assert bool((got[0][sl] != 0).any())
    for bad in ([(8, 4)], [(9, 4), (6, 4)], [(8, 0), (6, 4)], [(8,), (6, 4)]):
        with pytest.raises(ValueError):
            F.MuonPlan(views, 96, device, sides=bad)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("listed", [True, False])
def test_checkpoint_of_other_matrices(device, listed):
    """Refused before anything changes, with the list of matrices and, in a
    state that has none, by the moments; the same ones load either way."""
    saved = Muon(_arena(device), lr=0.5, exclude=("emb.w",))
    for seed in range(2):
        _grads(saved.arena, seed)
        saved.step()
    sd = saved.state_dict()
    assert sd["matrices"] == ["conv.w", "tall.w", "head.w"]
    if not listed:
        del sd["matrices"]
    for exclude in ((), ("emb.w", "head.w"), ("head.w",)):
        opt = Muon(_arena(device), lr=0.25, exclude=exclude)
        _grads(opt.arena, 5)
        opt.step()
        mom, m2 = opt.mom.clone(), opt.m2.clone()
        with pytest.raises(ValueError):
            opt.load_state_dict(sd)
        assert torch.equal(opt.mom, mom) and torch.equal(opt.m2, m2)
        assert int(opt.t) == 1 and opt.lr == 0.25
    opt = Muon(_arena(device), exclude=("emb.w",))
    opt.load_state_dict(sd)
    assert torch.equal(opt.mom, saved.mom) and int(opt.t) == 2 and opt.lr == 0.5
    with pytest.raises(ValueError):
        opt.load_state_dict({**sd, "m2": sd["m2"][:1]})
    assert torch.equal(opt.m2, saved.m2)


@pytest.mark.parametrize("device", DEVICES)
def test_arenas_that_share_memory(device):
    """One tensor in two places, or two that overlap, are refused before
    anything is written."""
    flat = torch.ones(5 * 64, device=device)
    own = [flat[i * 64:(i + 1) * 64] for i in range(4)]
    half = flat[256:].view(torch.bfloat16)[:64]
    plan = F.MuonPlan([(0, 4, 8)], 64, device)
    ranges = F.AdamRanges([(32, 64)], 64, device)
    step = torch.ones(1, dtype=torch.int32, device=device)

    def muon(t, mirror):
        F.muon_step(plan, *t, mirror, lr=0.1)

    def adam(t, mirror):
        F.adam_ranges(ranges, *t, mirror, 0.1, 0.9, 0.99, 1e-8, 0.0, step)

    for call, n in ((muon, 3), (adam, 4)):
        for i in range(n):
            for j in range(n):
                for bad in (own[j], flat[j * 64 + 8:j * 64 + 72]):
                    t = own[:n]
                    t[i] = bad
                    if i == j and bad is own[j] or i == n - 1 and j == n - 1:
                        continue
                    with pytest.raises(RuntimeError):
                        call(t, half)
            with pytest.raises(RuntimeError):
                call(own[:n], own[i].view(torch.bfloat16)[30:94])
        with pytest.raises(RuntimeError):
            call([*own[:n - 1], own[n - 1][:56]], half)
    assert bool((flat == 1).all())
    muon(own[:3], half)
    adam(own, half)
    assert bool((own[0][:32] != 1).any()) and bool((own[0][32:] != 1).all())
    if device == "cuda":
        with pytest.raises(RuntimeError):
            F.adam_ranges(ranges, *own, half, 0.1, 0.9, 0.99, 1e-8, 0.0,
                          step[:0])


def test_held_tensors():
    """All that a model's layers keep, whatever holds it."""
    m = build_textcnn("cpu", vocab=50, emb_dim=32, filters=64, layer_norm=True)
    ids, y = imdb_batch(4, seq_len=12, vocab=50, seed=0)
    m.train_step(ids, y)
    held = {id(t) for t in _held_tensors(m)}
    for lay in (m.ln_emb, m.ln_cat, *m.convs, m.fc):
        bufs = [t for t in lay._bufs.values() if isinstance(t, torch.Tensor)]
        assert bufs and all(id(t) in held for t in bufs)
    assert all(id(t) in held for t in (m.arena.master, m.arena.mirror,
                                       m.arena.grad, m.emb._out, m.loss_sum))


@pytest.mark.gpu
def test_predictions_between_captured_steps():
    """Another batch size between replays: the layers' buffers are replaced, and
    the captured step neither loses its own nor writes to new tensors."""
    gen = torch.Generator().manual_seed(9)
    x = torch.randn(96, 48, generator=gen).bfloat16().cuda()
    y = torch.randint(0, 10, (96,), generator=gen).cuda()
    twin, m = _network("cuda"), _network("cuda")
    eager = Trainer(twin, make_muon(twin, exclude=("fc2.w",)), "cuda")
    graph = Trainer(m, make_muon(m, exclude=("fc2.w",)), "cuda", use_graph=True)
    graph.step_async(x, y)          # warms up with three steps and captures
    for _ in range(3):
        eager.step_async(x, y)
    assert graph._graph is not None
    own = {t.data_ptr() for t in graph._graph_held}
    m.predict(x[:40])
    new = [torch.full_like(t, 3) for t in graph._graph_held for _ in range(3)]
    assert not own & {t.data_ptr() for t in new}
    for n in (40, 17, 96):
        graph.step_async(x, y)
        eager.step_async(x, y)
        assert torch.equal(m.predict(x[:n]), twin.predict(x[:n]))
        assert torch.equal(m.arena.master, twin.arena.master)
    assert all(bool((t == 3).all()) for t in new)
