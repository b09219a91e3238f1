"""The orthogonalised update and the optimizer built on it against float64: odd sizes, types, strides, batches, ranks; refusals.

Tolerances: the products run on f16 operands.  ``_emulated`` repeats the iteration in float64 with exactly the kernel's three roundings a
step (X, and A and B beside their diagonals, to f16; X itself unrounded), which says for each input how far those carry the result; the kernel adds float32 sums
and other signs of the same roundings, for which the bound is twice that, plus half a step of the bf16 result."""

import contextlib
import copy
import ctypes
import math
import os
import pickle
import subprocess

import pytest
import torch

from mmlearn_amd.optim import NS_COEFFICIENTS, Muon, orthogonalize
from oracle import tower_oracle as oracle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _emulated(g, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    s = 2.0 ** int(math.log2(max(g.shape)) / 2)

    def r(t):
        return (t * s).to(torch.float16).double() / s

    def parts(t):      # the diagonal exact, the rest rounded
        d = torch.diag(t.diagonal())
        return d, r(t - d)

    x = x / (x.square().sum().sqrt() + eps)
    for _ in range(steps):
        h = r(x)
        da, ea = parts(h @ h.T)
        db, eb = parts(b * (da + ea) + c * (da + ea) @ (da + ea))
        x = a * x + db @ x + eb @ h
    return x.T if tall else x


def _tolerance(g, want, **how):
    """(of the 2-norm, of the largest element)"""
    off = (_emulated(g, **how) - want).norm().item()
    rms = 2 * off / math.sqrt(want.numel())
    return 2 * off + 2.0 ** -8 * want.norm().item() + 1e-6, 16 * rms + 2.0 ** -8 * want.abs().max().item() + 1e-6


def _matrix(rows, cols, kind, g):
    if kind == "low rank":     # a few strong directions over faint noise
        k = max(1, min(rows, cols) // 16)
        return torch.randn(rows, k, generator=g) @ torch.randn(k, cols, generator=g) + 0.05 * torch.randn(rows, cols, generator=g)
    if kind == "one":
        return torch.outer(torch.randn(rows, generator=g), torch.randn(cols, generator=g))
    if kind == "spiked":       # one entry is nearly everything
        x = 1e-3 * torch.randn(rows, cols, generator=g)
        x[rows // 2, cols // 2] = 1.0
        return x
    return torch.randn(rows, cols, generator=g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,cols,kind", [
    (1, 1, "noise"), (1, 7, "noise"), (5, 3, "noise"), (64, 64, "low rank"), (65, 201, "noise"), (201, 65, "low rank"), (128, 128, "noise"),
    (129, 300, "spiked"), (300, 129, "one"), (256, 1000, "low rank"), (640, 257, "noise"), (33, 2100, "noise"),
])
def test_against_float64(rows, cols, kind, dtype):
    g = torch.Generator().manual_seed(rows * 1000 + cols)
    x = (1e-3 * _matrix(rows, cols, kind, g)).to(getattr(torch, dtype))
    got = orthogonalize(x.cuda())
    assert got.dtype == torch.bfloat16 and got.shape == x.shape and got.is_contiguous()
    want = oracle.orthogonalize(x)
    d = got.double().cpu() - want
    norm, most = _tolerance(x, want)
    assert d.norm() <= norm and d.abs().max() <= most, (d.norm().item() / want.norm().item(), norm / want.norm().item())


@pytest.mark.gpu
def test_batches_strides_and_neighbours():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 40, 90, generator=g)
    x[0, 1] = 0
    x[1, 1, 3, 4] = float("nan")
    x[1, 2, 0, 0] = float("inf")
    wide = torch.zeros(2, 3, 44, 200)
    wide[:, :, 2:42, 10:190:2] = x
    for t in (x.cuda(), wide.cuda()[:, :, 2:42, 10:190:2], x.transpose(2, 3).contiguous().cuda().transpose(2, 3), x.transpose(0, 1).contiguous().cuda().transpose(0, 1)):
        got = orthogonalize(t).double().cpu()
        assert not got[0, 1].any() and got[1, 1].isnan().all() and got[1, 2].isnan().all()
        for i, j in ((0, 0), (0, 2), (1, 0)):
            want = oracle.orthogonalize(x[i, j])
            assert (got[i, j] - want).norm() <= _tolerance(x[i, j], want)[0]
    many = torch.randn(131, 9, 20, generator=g)     # more matrices than one launch takes
    got = orthogonalize(many.cuda()).double().cpu()
    for i in (0, 63, 64, 127, 128, 130):
        want = oracle.orthogonalize(many[i])
        assert (got[i] - want).norm() <= _tolerance(many[i], want)[0]
    assert orthogonalize(torch.zeros(0, 4, 5, device="cuda")).shape == (0, 4, 5) and orthogonalize(torch.zeros(4, 0, device="cuda")).shape == (4, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("count,rows,cols", [(22, 384, 640), (40, 640, 384), (64, 1280, 100), (64, 640, 640), (64, 500, 510), (3, 130, 4000)])
def test_batches_that_fill_the_chip_differently(count, rows, cols):
    """Few tiles, some for every CU, many, and 256 x 256 ones."""
    x = torch.randn(count, rows, cols, generator=torch.Generator().manual_seed(count))
    x[count // 2] *= 1e4
    got = orthogonalize(x.cuda()).double().cpu()
    for i in (0, count // 2, count - 1):
        want = oracle.orthogonalize(x[i])
        norm, most = _tolerance(x[i], want)
        d = got[i] - want
        assert d.norm() <= norm and d.abs().max() <= most, (i, d.norm().item() / want.norm().item())


@pytest.mark.gpu
@pytest.mark.parametrize("steps,coefficients", [(1, NS_COEFFICIENTS), (2, (1.875, -1.25, 0.375)), (8, (1.875, -1.25, 0.375)), (6, (1.5, -0.5, 0.0))])
def test_other_iterations(steps, coefficients):
    x = torch.randn(70, 140, generator=torch.Generator().manual_seed(3))
    want = oracle.orthogonalize(x, steps, coefficients, 1e-3)
    d = orthogonalize(x.cuda(), steps, coefficients, 1e-3).double().cpu() - want
    assert d.norm() <= _tolerance(x, want, steps=steps, coefficients=coefficients, eps=1e-3)[0]


@pytest.mark.gpu
def test_scale_of_the_input_does_not_matter():
    x = torch.randn(96, 200, generator=torch.Generator().manual_seed(3)).cuda()
    want = orthogonalize(x)
    for s in (2.0 ** 100, 2.0 ** -10):
        got = orthogonalize(x * s)     # (|x| 2^-10 is 0.13, so eps takes 8e-7 of it)
        assert (got.double() - want.double()).norm() <= 2.0 ** -8 * want.double().norm()


@pytest.mark.gpu
def test_repeatable_captured_and_on_two_streams():
    x = torch.randn(3, 200, 333, generator=torch.Generator().manual_seed(5)).cuda()
    want = orthogonalize(x)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(orthogonalize(x))
    for s in (s1, s2):
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(t, want) for t in got)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = orthogonalize(x)
    for _ in range(3):
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want) and torch.equal(orthogonalize(x), want)


def _muon_oracle(w, buf, g, lr, wd, mu, nesterov, match):
    buf = mu * buf + g
    u = g + mu * buf if nesterov else buf
    adjust = 0.2 * math.sqrt(max(w.shape)) if match else math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
    o = oracle.orthogonalize(u)
    return w * (1 - lr * wd) - lr * adjust * o, buf, lr * adjust * _tolerance(u, o)[1]


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov,match", [(True, False), (False, True)])
def test_muon_steps(nesterov, match):
    g = torch.Generator().manual_seed(9)
    shapes = [(64, 200), (200, 64), (64, 200), (130, 130), (7, 5)]
    start = [0.1 * torch.randn(*s, generator=g) for s in shapes]
    params = [torch.nn.Parameter(t.cuda()) for t in start]
    idle = torch.nn.Parameter(torch.ones(3, 3, device="cuda"))
    opt = Muon([*params, idle], lr=0.02, weight_decay=0.1, momentum=0.9, nesterov=nesterov, adjust_lr_fn="match_rms_adamw" if match else None)
    want, bufs, slack = [t.double() for t in start], [torch.zeros(s, dtype=torch.float64) for s in shapes], [0.0] * len(shapes)
    for step in range(3):
        for i, p in enumerate(params):
            grad = 1e-2 * torch.randn(*shapes[i], generator=g)
            p.grad = grad.cuda() if step != 1 else grad.t().contiguous().cuda().t()     # one step with transposed gradients
            want[i], bufs[i], tol = _muon_oracle(want[i], bufs[i], grad.double(), 0.02, 0.1, 0.9, nesterov, match)
            slack[i] += tol
        before = [p._version for p in params]
        opt.step()
        for i, p in enumerate(params):
            assert (p.detach().double().cpu() - want[i]).abs().max() <= slack[i] + 4 * 2.0 ** -24, (step, shapes[i])
            b = opt.state[p]["momentum_buffer"].double().cpu()
            assert (b - bufs[i]).abs().max() <= (step + 1) * 2.0 ** -23 * bufs[i].abs().max()
        assert all(p._version > v for p, v in zip(params, before))
    assert torch.equal(idle.detach(), torch.ones_like(idle)) and idle not in opt.state
    # the state travels
    other = Muon([torch.nn.Parameter(p.detach().clone()) for p in params] + [idle], lr=0.02)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))     # (a state dict holds the tensors themselves)
    for p, r in zip(params, other.param_groups[0]["params"]):
        r.grad = p.grad
    opt.step()
    other.step()
    assert all(torch.equal(p, r) for p, r in zip(params, other.param_groups[0]["params"]))


@pytest.mark.gpu
def test_a_captured_muon_step_follows_the_learning_rate(monkeypatch):
    def fresh():
        p = torch.nn.Parameter(torch.linspace(-1, 1, 64 * 150).sin().view(64, 150).cuda())
        p.grad = torch.linspace(-3, 2, 64 * 150).cos().view(64, 150).cuda()
        return p

    p, r = fresh(), fresh()
    opt, eager = Muon([p], lr=0.01, capturable=True), Muon([r], lr=0.01)
    opt.step()
    eager.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for lr in (0.01, 0.03, 0.005):
        opt.lr_device().fill_(lr)
        eager.param_groups[0]["lr"] = lr
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        # the rate passes through a float32 word on one side
        assert (p.detach() - r.detach()).abs().max() <= 2.0 ** -22 * (1 + r.detach().abs().max())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="eager step"):
        Muon([fresh()], capturable=True).step()


def test_struct_layout_matches_header():
    from mmlearn_amd import _lib

    src = '#include <stdio.h>\n#include "mmlearn_hip.h"\nint main(){printf("%zu %zu", sizeof(mmk_newton_schulz_args), offsetof(mmk_newton_schulz_args, weight_decay));return 0;}'
    exe = "/tmp/_mmk_ns_sizeof"
    subprocess.run(["gcc", "-x", "c", "-", "-I", os.path.join(ROOT, "include"), "-o", exe], input=src, text=True, check=True)
    size, last = map(int, subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split())
    assert ctypes.sizeof(_lib.NewtonSchulz) == size and _lib.NewtonSchulz.weight_decay.offset == last


def test_refusals(monkeypatch):
    from mmlearn_amd import optim as O

    with pytest.raises(RuntimeError, match="no CPU fallback"):
        orthogonalize(torch.zeros(4, 4))
    monkeypatch.setattr(O, "require_gpu", lambda *a: None)
    monkeypatch.setattr(O.K, "newton_schulz", lambda *a: pytest.fail("reached the kernel"))
    x = torch.zeros(4, 6)
    for bad in (dict(update=x[0]), dict(update=x.double()), dict(update=torch.zeros(1, 32769)), dict(steps=0), dict(steps=33), dict(steps=2.0), dict(coefficients=(1.0, 2.0)),
                dict(coefficients=(1.0, float("nan"), 0.0)), dict(coefficients=(1.0, 100.0, 0.0)), dict(eps=0.0), dict(eps=float("inf"))):
        with pytest.raises(ValueError):
            orthogonalize(**{"update": x, **bad})
    w = torch.nn.Parameter(torch.zeros(3, 3))
    for bad in (dict(lr=-1.0), dict(lr=float("nan")), dict(momentum=1.0), dict(weight_decay=-0.1), dict(ns_steps=0), dict(eps=0.0), dict(adjust_lr_fn="other"), dict(ns_coefficients=(1.0,))):
        with pytest.raises(ValueError):
            Muon([w], **bad)
    for shape in ((3,), (2, 3, 4), ()):
        with pytest.raises(ValueError, match="matrices"):
            Muon([torch.nn.Parameter(torch.zeros(shape))])
    for p in (torch.nn.Parameter(torch.zeros(3, 3).bfloat16()), torch.nn.Parameter(torch.zeros(3, 4).t())):
        p.grad = torch.zeros_like(p)
        with pytest.raises(RuntimeError, match="dense contiguous f32"):
            Muon([p]).step()


def test_forward_mode_derivatives_are_refused(monkeypatch):
    from torch.autograd import forward_ad as fw

    from mmlearn_amd import optim as O

    monkeypatch.setattr(O, "require_gpu", lambda *a: None)
    monkeypatch.setattr(O._lib, "on_device_of", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(O.K, "newton_schulz", lambda *a: None)
    x = torch.zeros(4, 6)
    with fw.dual_level():
        assert orthogonalize(x).shape == (4, 6)
        with pytest.raises(NotImplementedError, match="forward"):
            orthogonalize(fw.make_dual(x, x))


def _torch_muon_state(start, grads, **how):
    """A state of ``torch.optim.Muon`` after steps on the CPU, and the weights they lead to."""
    params = [torch.nn.Parameter(t.clone()) for t in start]
    opt = torch.optim.Muon(params, **how)
    for gs in grads:
        for p, g in zip(params, gs):
            p.grad = g.clone()
        opt.step()
    return opt, params


@pytest.mark.parametrize("momentum", [0.95, 0.0])
def test_a_state_of_torch_muon_is_converted(momentum):
    g = torch.Generator().manual_seed(21)
    start = [torch.randn(5, 7, generator=g), torch.randn(6, 4, generator=g)]
    grads = [[torch.randn(t.shape, generator=g) for t in start] for _ in range(4)]
    theirs, params = _torch_muon_state(start, grads, lr=0.02, momentum=momentum)
    before = [theirs.state[p]["momentum_buffer"].clone() for p in params]
    idle = torch.nn.Parameter(torch.zeros(2, 2))
    mine = [torch.nn.Parameter(p.detach().clone()) for p in params]
    opt = Muon(mine, lr=0.5, capturable=True)
    opt.load_state_dict(theirs.state_dict())
    for i, p in enumerate(mine):
        m = torch.zeros(start[i].shape, dtype=torch.float64)
        for gs in grads:
            m = momentum * m + gs[i].double()
        # theirs: a subtraction, a product and a sum in float32 a step; then the factor 1 / (1 - momentum) = 20, itself of float32
        assert (opt.state[p]["momentum_buffer"].double() - m).abs().max() <= 4 * 4 * 2.0 ** -24 * m.abs().max() / (1 - momentum)
        assert torch.equal(theirs.state[params[i]]["momentum_buffer"], before[i])
    assert opt.param_groups[0]["lr"] == 0.02 and opt.param_groups[0]["capturable"] is True
    mixed = Muon([{"params": [torch.nn.Parameter(p.detach().clone()) for p in params], "capturable": True}])     # (a group's own choice)
    mixed.load_state_dict(theirs.state_dict())
    assert mixed.param_groups[0]["capturable"] is True
    # a state of this class stays as it is
    other = Muon([torch.nn.Parameter(p.detach().clone()) for p in params] + [idle])
    sd = opt.state_dict()
    sd["param_groups"][0]["params"].append(2)
    other.load_state_dict(sd)
    for p, r in zip(mine, other.param_groups[0]["params"]):
        assert torch.equal(opt.state[p]["momentum_buffer"], other.state[r]["momentum_buffer"])
    Muon([idle]).load_state_dict(torch.optim.Muon([idle]).state_dict())     # (nothing in it yet)
    with pytest.raises(ValueError, match="momentum"):
        Muon([idle]).load_state_dict(torch.optim.Muon([idle], momentum=1.0).state_dict())
    for how in (dict(ns_steps=40), dict(eps=1e-50)):     # refused here, not in the middle of a step
        with pytest.raises(ValueError):
            Muon([idle]).load_state_dict(torch.optim.Muon([idle], **how).state_dict())


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov", [True, False])
def test_continues_from_a_state_of_torch_muon(nesterov):
    g = torch.Generator().manual_seed(22)
    start = [0.1 * torch.randn(40, 60, generator=g), 0.1 * torch.randn(130, 70, generator=g)]
    grads = [[1e-2 * torch.randn(t.shape, generator=g) for t in start] for _ in range(4)]
    theirs, params = _torch_muon_state(start, grads, lr=0.02, momentum=0.95, nesterov=nesterov, weight_decay=0.0)
    mine = [torch.nn.Parameter(p.detach().clone().cuda()) for p in params]
    opt = Muon(mine)
    opt.load_state_dict(theirs.state_dict())
    last = [1e-2 * torch.randn(t.shape, generator=g) for t in start]
    for p, x in zip(mine, last):
        p.grad = x.cuda()
    opt.step()
    for i, p in enumerate(mine):
        buf = torch.zeros(start[i].shape, dtype=torch.float64)
        for gs in grads:
            buf = 0.95 * buf + gs[i].double()
        want, _, tol = _muon_oracle(params[i].detach().double(), buf, last[i].double(), 0.02, 0.0, 0.95, nesterov, False)
        assert (p.detach().double().cpu() - want).abs().max() <= tol + 4 * 2.0 ** -24


def _on_the_host(monkeypatch, calls):
    """Muon's host side without a GPU: every launch is written down."""
    from mmlearn_amd import optim as O

    monkeypatch.setattr(O, "require_gpu", lambda *a: None)
    monkeypatch.setattr(O._lib, "on_device_of", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(O.K, "newton_schulz", lambda src, dst, rows, cols, *a: calls.append((rows, cols, a[-4], None if a[-1] is None else a[-1].item())))


@pytest.mark.parametrize("tensor", [True, False])
def test_capturable_eager_steps_follow_a_learning_rate_filled_in_place(monkeypatch, tensor):
    calls = []
    _on_the_host(monkeypatch, calls)
    p = torch.nn.Parameter(torch.zeros(3, 4))
    opt = Muon([p], lr=torch.tensor(0.5) if tensor else 0.5, capturable=True)
    for lr in (0.5, 0.25, 0.25, 0.125):
        if tensor:
            opt.param_groups[0]["lr"].fill_(lr)
        else:
            opt.param_groups[0]["lr"] = lr
        p.grad = torch.ones_like(p)
        opt.step()
        assert calls[-1][3] == lr and opt.lr_device().item() == lr
    plain = Muon([p], lr=torch.tensor(0.5))
    plain.param_groups[0]["lr"].fill_(0.25)
    plain.step()
    assert calls[-1][2:] == (0.25, None)


def test_a_refused_step_moves_nothing(monkeypatch):
    calls = []
    _on_the_host(monkeypatch, calls)
    good = torch.nn.Parameter(torch.zeros(3, 4))
    for other in (torch.nn.Parameter(torch.zeros(4, 5).t()), torch.nn.Parameter(torch.zeros(4, 5).bfloat16()), torch.nn.Parameter(torch.zeros(32768, 1))):
        for p in (good, other):
            p.grad = torch.ones_like(p)
        opt = Muon([{"params": [good]}, {"params": [other]}])
        if other.shape == (32768, 1):
            opt.step()
            assert [c[:2] for c in calls] == [(3, 4), (32768, 1)]
            continue
        with pytest.raises(RuntimeError, match="dense contiguous f32"):
            opt.step()
        assert not calls and not opt.state
    # a matrix too wide for the kernels is refused where it is added, and leaves nothing behind
    for shape, why in (((32769, 1), "32768"), ((2, 40000), "32768"), ((3,), "matrices")):
        with pytest.raises(ValueError, match=why):
            opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(shape))]})
        assert len(opt.param_groups) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(20, 30), (130, 260)])
def test_zeros_stay_zero_at_the_smallest_eps(shape):
    x = torch.zeros(2, *shape, device="cuda")
    x[1] = 1.0
    got = orthogonalize(x, eps=2.0 ** -126)
    assert not got[0].any() and torch.isfinite(got).all()


def test_an_eps_that_float32_cannot_divide_by_is_refused(monkeypatch):
    from mmlearn_amd import _lib
    from mmlearn_amd import optim as O

    monkeypatch.setattr(O, "require_gpu", lambda *a: None)
    monkeypatch.setattr(O.K, "newton_schulz", lambda *a: pytest.fail("reached the kernel"))
    for eps in (1e-39, 1e-60, 2.0 ** -149):
        with pytest.raises(ValueError, match="eps"):
            orthogonalize(torch.zeros(4, 6), eps=eps)
        with pytest.raises(ValueError, match="eps"):
            Muon([torch.nn.Parameter(torch.zeros(3, 3))], eps=eps)
        args = _lib.NewtonSchulz()
        args.count, args.rows, args.cols, args.steps, args.eps = 0, 4, 6, 5, eps
        assert _lib.lib().mmk_newton_schulz(ctypes.byref(args), None, None) != 0


@pytest.mark.gpu
@pytest.mark.parametrize("count,rows,cols", [(3, 300, 129), (3, 129, 301), (22, 384, 640), (40, 640, 380), (64, 500, 510), (70, 130, 140), (2, 512, 5000)])
def test_muon_steps_of_batches(count, rows, cols):
    """Two steps (momenta that are not zero) of several equal matrices at once: few tiles, some for every CU, many, 256 x 256 ones, more matrices than
    one launch takes; columns that fit no vector."""
    g = torch.Generator().manual_seed(count)
    start = 0.1 * torch.randn(count, rows, cols, generator=g)
    params = [torch.nn.Parameter(t.cuda()) for t in start]
    opt = Muon(params, lr=0.02, weight_decay=0.1, momentum=0.9)
    which = sorted({0, count // 2, count - 1})
    want = {i: start[i].double() for i in which}
    bufs, slack = {i: torch.zeros(rows, cols, dtype=torch.float64) for i in which}, dict.fromkeys(which, 0.0)
    for step in range(2):
        grads = 1e-2 * torch.randn(count, rows, cols, generator=g)
        grads[count // 2] *= 1e3
        for p, x in zip(params, grads):
            p.grad = x.cuda()
        opt.step()
        for i in which:
            want[i], bufs[i], tol = _muon_oracle(want[i], bufs[i], grads[i].double(), 0.02, 0.1, 0.9, True, False)
            slack[i] += tol
            assert (params[i].detach().double().cpu() - want[i]).abs().max() <= slack[i] + 4 * 2.0 ** -24, (step, i)
            b = opt.state[params[i]]["momentum_buffer"].double().cpu()
            assert (b - bufs[i]).abs().max() <= (step + 1) * 2.0 ** -23 * bufs[i].abs().max(), (step, i)


def test_momenta_and_weights_go_together():
    from mmlearn_amd import _lib

    at = (ctypes.c_void_p * 1)(1 << 20)
    for momenta, weights in ((None, 1), (ctypes.cast(at, ctypes.c_void_p), 0)):
        p = _lib.NewtonSchulz()
        p.src = p.dst = ctypes.cast(at, ctypes.c_void_p)
        p.count, p.rows, p.cols, p.steps, p.eps, p.momenta, p.weights = 1, 8, 8, 5, 1e-7, momenta, weights
        assert _lib.lib().mmk_newton_schulz(ctypes.byref(p), None, None) == -1 and b"momenta and weights" in _lib.lib().mmk_last_error()


def test_copies_of_the_optimizer_work(monkeypatch):
    calls = []
    _on_the_host(monkeypatch, calls)
    p = torch.nn.Parameter(torch.zeros(3, 4))
    opt = Muon([p], lr=0.5, capturable=True)
    p.grad = torch.ones_like(p)
    opt.step()
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        other.param_groups[0]["lr"] = 0.25
        other.param_groups[0]["params"][0].grad = torch.ones_like(p)
        other.step()
        assert calls[-1][3] == 0.25 and other.lr_device().item() == 0.25 and opt.lr_device().item() == 0.5
    word = opt.lr_device()
    opt.load_state_dict(copy.deepcopy(opt.state_dict()))
    opt.step()
    assert opt.lr_device() is word and word.item() == 0.5     # (a captured step reads this word)
