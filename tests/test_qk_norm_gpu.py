"""Per-head norm of queries and keys with the position rotation against its float64 definition: layouts, odd sizes, strides, types,
positions; the gradients against autograd of the definition and against differences; graphs, streams; the refusals."""

import pytest
import torch

from mmlearn_amd.attention import qk_norm_rotary, rotary_table
from oracle import tower_oracle as oracle

EPS = 1e-6


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _view(x, kind):
    """The same values behind other strides."""
    if kind == "packed":      # heads of a wider projection
        wide = torch.full((*x.shape[:2], x.shape[2] + 3, x.shape[3]), float("nan"), dtype=x.dtype, device=x.device)
        wide[:, :, 1:1 + x.shape[2]] = x
        return wide[:, :, 1:1 + x.shape[2]]
    if kind == "heads first":
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if kind == "odd":         # rows that start off any 16-byte border
        wide = torch.full((*x.shape[:3], x.shape[3] + 1), float("nan"), dtype=x.dtype, device=x.device)
        wide[..., 1:] = x
        return wide[..., 1:]
    return x


def _close(got, want, terms, dtype, extra=8):
    """got within half a step of the type of want, plus `extra` float32 roundings of the terms it is summed from."""
    bound = _half_step(dtype) * want.abs() * 1.0001 + extra * 2.0 ** -24 * terms
    bad = (got.double().cpu() - want).abs() - bound
    assert bad.max().item() <= 0 if bad.numel() else True, (bad.max().item(), want.abs().max().item())


CASES = [
    # B, L, H, Hk, D, rot, interleaved, dtype, weights, positions, strides
    (1, 1, 1, 1, 64, 64, False, "bfloat16", "same", None, "plain"),
    (2, 5, 12, 12, 64, 64, False, "bfloat16", "f32", "row", "packed"),
    (3, 7, 8, 2, 128, 128, True, "bfloat16", "same", "batch", "packed"),
    (2, 33, 4, 1, 128, 64, False, "float16", "f32", "batch64", "heads first"),
    (2, 9, 3, 3, 80, 40, False, "float32", "same", "row64", "plain"),
    (1, 11, 5, 1, 96, 0, False, "float16", "same", None, "plain"),
    (2, 4, 3, 2, 2, 2, True, "float32", "same", None, "plain"),
    (2, 3, 2, 1, 254, 254, False, "bfloat16", "same", "row", "odd"),
    (1, 3, 2, 2, 256, 254, True, "float32", "none", "batch", "odd"),
    (2, 6, 3, 1, 32, 10, False, "bfloat16", "none", "row", "odd"),
    (2, 6, 3, 1, 6, 4, True, "float16", "q", "row", "plain"),
    (4, 197, 12, 12, 64, 64, False, "bfloat16", "f32", None, "packed"),
    (1, 2049, 16, 4, 128, 64, True, "bfloat16", "same", "row", "packed"),
]


def _inputs(case, seed=0):
    B, L, H, Hk, D, rot, ilv, dtype, weights, positions, strides = case
    g = torch.Generator().manual_seed(seed)
    dt = getattr(torch, dtype)
    q, k = (2.0 * torch.randn(B, L, h, D, generator=g) for h in (H, Hk))
    q[0, 0, 0] = 0.0          # a head of zeros: eps decides
    k[-1, -1, -1] *= 1e-3
    q, k = (_view(x.to(dt).cuda(), strides) for x in (q, k))
    wdt = torch.float32 if weights == "f32" else dt
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g)).to(wdt).cuda() for _ in range(2))
    if weights == "none":
        qw = kw = None
    if weights == "q":
        kw = None
    table = rotary_table(5000, rot, device="cuda") if rot else None
    pos = None
    if positions:
        pos = torch.randint(0, 5000, (B, L) if "batch" in positions else (L,), generator=g)
        pos = pos.to(torch.int64 if "64" in positions else torch.int32).cuda()
    dq, dk = (torch.randn(B, L, h, D, generator=g).to(dt).cuda() for h in (H, Hk))
    return q, k, qw, kw, table, pos, ilv, dq, dk


def _oracle(x, w, table, pos, ilv, dy):
    x = x.detach().double().cpu().requires_grad_(True)
    w = None if w is None else w.detach().double().cpu().requires_grad_(True)
    y = oracle.qk_norm_rotary(x, w, None if table is None else table.double().cpu(), None if pos is None else pos.cpu(), ilv, EPS)
    leaves = (x,) if w is None else (x, w)
    grads = torch.autograd.grad(y, leaves, dy.double().cpu())
    return y.detach(), grads[0], grads[1] if w is not None else None


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_against_float64(case):
    q, k, qw, kw, table, pos, ilv, dq, dk = _inputs(case)
    dt = q.dtype
    leaves = [t.detach().requires_grad_(True) for t in (q, k)] + [None if w is None else w.requires_grad_(True) for w in (qw, kw)]
    got = qk_norm_rotary(*leaves, rotary=table, positions=pos, interleaved=ilv, eps=EPS)
    assert all(y.is_contiguous() and y.dtype == dt for y in got)
    real = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip("q k qw kw".split(), leaves) if t is not None], torch.autograd.grad(got, real, (dq, dk))))
    for n, x, w, y, dy in (("q", q, qw, got[0], dq), ("k", k, kw, got[1], dk)):
        want, dx, dw = _oracle(x, w, table, pos, ilv, dy)
        # a rotated value is the sum of two products, each after a sum of squares, a root, a reciprocal and two products: 8 roundings of
        # the row's largest value cover them (sums of D <= 256 squares in vectors and a tree add at most 16 half steps under the root)
        rows = want.abs().amax(-1, keepdim=True)
        _close(y, want, rows, dt, 16)
        # dx is the difference of g w and n mean(g w n), times the reciprocal root
        rstd = (x.double().cpu().square().mean(-1, keepdim=True) + EPS).rsqrt()
        gmax = (dy.double().cpu().norm(dim=-1, keepdim=True)) * (1 if w is None else w.detach().double().cpu().abs().max())
        _close(grads[n], dx, rstd * gmax, dt, 32)
        if w is not None:
            # dw: per-lane sums over rows, then over groups and workgroups; every term carries the roundings of g and n
            n_hat = (x.double().cpu() * rstd).abs()
            terms = (dy.double().cpu().norm(dim=-1, keepdim=True) * n_hat).sum((0, 1, 2))
            rows_n = x.shape[0] * x.shape[1] * x.shape[2]
            _close(grads[n + "w"], dw, terms, w.dtype, 32 + min(rows_n, 400))


@pytest.mark.gpu
def test_gradients_against_differences():
    q, k, qw, kw, table, pos, ilv, dq, dk = _inputs((1, 3, 2, 1, 16, 8, False, "float32", "same", "row", "plain"), 3)
    q[0, 0, 0] = 1.0
    leaves = [t.detach().requires_grad_(True) for t in (q, k, qw, kw)]
    y = qk_norm_rotary(*leaves, rotary=table, positions=pos)
    grads = torch.autograd.grad(y, leaves, (dq, dk))
    g = torch.Generator().manual_seed(1)
    for n, leaf in enumerate(leaves):
        d = torch.randn(leaf.shape, generator=g).cuda()
        d /= d.norm()
        # sqrt(D) x / |x| along a unit direction: the third derivative is at most 15 sqrt(D) / |x|^3, so the central difference is off by
        # h^2 / 6 of that.  The last key head is a thousand times smaller than the others: h goes by the smallest row (a fixed 2^-6 would
        # be larger than that row itself).  The weights enter linearly.  The float32 outputs, up to sqrt(D) w each with about four
        # roundings, are differenced over 2 h.
        x_min = leaf.detach().norm(dim=-1).min().item() if n < 2 else None
        h = x_min / 64 if n < 2 else 2.0 ** -6

        def f(t):
            a = [x.detach() for x in leaves]
            a[n] = a[n] + t * d
            out = qk_norm_rotary(*a, rotary=table, positions=pos)
            return (out[0].double() * dq).sum().item() + (out[1].double() * dk).sum().item()

        want = (f(h) - f(-h)) / (2 * h)
        scale = (dq.norm() + dk.norm()).item() * max(1.0, qw.abs().max().item(), kw.abs().max().item())
        truncation = 15 * 4 * h * h / 6 / x_min ** 3 if n < 2 else 0.0
        assert abs((grads[n].double() * d).sum().item() - want) < scale * (truncation + 4 * 4 * 2.0 ** -24 / h)


@pytest.mark.gpu
def test_rows_of_nothing_and_of_one_side():
    w = torch.ones(64, device="cuda", requires_grad=True)
    for shape_q, shape_k in (((2, 0, 3, 64), (2, 0, 1, 64)), ((0, 4, 3, 64), (0, 4, 1, 64)), ((2, 4, 0, 64), (2, 4, 2, 64)), ((2, 4, 2, 64), (2, 4, 0, 64))):
        q, k = torch.randn(shape_q, device="cuda", requires_grad=True), torch.randn(shape_k, device="cuda", requires_grad=True)
        y = qk_norm_rotary(q, k, w, w)
        grads = torch.autograd.grad(y, (q, k, w), [torch.ones_like(t) for t in y])
        assert y[0].shape == shape_q and y[1].shape == shape_k and grads[0].shape == shape_q and grads[1].shape == shape_k
        assert torch.isfinite(grads[2]).all() and (bool(grads[2].any()) == (q.numel() + k.numel() > 0))


@pytest.mark.gpu
def test_a_position_outside_the_table_is_loud_and_harmless():
    table = rotary_table(16, 64, device="cuda")
    q, k = torch.randn(1, 4, 2, 64, device="cuda"), torch.randn(1, 4, 1, 64, device="cuda")
    pos = torch.tensor([3, -1, 16, 15], dtype=torch.int64, device="cuda")
    y, z = qk_norm_rotary(q, k, rotary=table, positions=pos)
    bad = torch.tensor([False, True, True, False], device="cuda")
    assert y[0, bad].isnan().all() and z[0, bad].isnan().all() and y[0, ~bad].isfinite().all() and z[0, ~bad].isfinite().all()


@pytest.mark.gpu
def test_broadcast_operands_and_one_weight_for_both():
    g = torch.Generator().manual_seed(5)
    one = torch.randn(1, 1, 1, 64, generator=g).cuda().requires_grad_(True)
    k = torch.randn(2, 3, 2, 64, generator=g).cuda().requires_grad_(True)
    w = torch.randn(64, generator=g).cuda().requires_grad_(True)
    y = qk_norm_rotary(one.expand(2, 3, 4, 64), k, w, w)
    dy = [torch.randn(t.shape, generator=g).cuda() for t in y]
    grads = torch.autograd.grad(y, (one, k, w), dy)
    a, b, c = (t.detach().double().cpu().requires_grad_(True) for t in (one, k, w))
    want = torch.autograd.grad([oracle.qk_norm_rotary(x, c, None, None, False, EPS) for x in (a.expand(2, 3, 4, 64), b)], (a, b, c),
                               [t.double().cpu() for t in dy])
    for x, z in zip(grads, want):
        # 24 rows are summed outside and inside; 64 roundings of the largest gradient cover them
        assert (x.double().cpu() - z).abs().max() <= 64 * 2.0 ** -24 * z.abs().max() * 24


@pytest.mark.gpu
def test_bitwise_repeatable_captured_and_on_another_stream():
    q, k, qw, kw, table, pos, ilv, dq, dk = _inputs((4, 197, 12, 4, 64, 64, False, "bfloat16", "f32", "batch", "packed"))
    leaves = [t.detach().requires_grad_(True) for t in (q, k, qw, kw)]

    def step():
        # detached: an output that keeps its autograd graph keeps the leaves' gradient nodes on the stream of that pass, and a backward
        # captured on another stream then waits for a stream outside the capture, which ends the process
        y = qk_norm_rotary(*leaves, rotary=table, positions=pos)
        grads = torch.autograd.grad(y, leaves, (dq, dk))
        return [t.detach() for t in (*y, *grads)]

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        for t in held:
            t.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held))
        assert all(torch.equal(a, b) for a, b in zip(want, step()))


def test_refusals(monkeypatch):
    """Checked on the CPU: the device test is the first of them, so it is taken out of the way."""
    from mmlearn_amd import attention as A

    with pytest.raises(RuntimeError, match="no CPU fallback"):
        qk_norm_rotary(torch.zeros(1, 1, 1, 64), torch.zeros(1, 1, 1, 64))
    monkeypatch.setattr(A.K, "require_gpu", lambda *a: None)
    monkeypatch.setattr(A._QKNormRotary, "apply", lambda *a: pytest.fail("reached the kernel"))
    q, k, w = torch.zeros(2, 3, 4, 64), torch.zeros(2, 3, 2, 64), torch.ones(64)
    table = rotary_table(8, 64)
    for bad in (
        dict(q=q[0]), dict(k=k[:1]), dict(k=k[..., :32]), dict(k=k.bfloat16()), dict(q=q.double(), k=k.double()),
        dict(q=q[..., :63], k=k[..., :63]), dict(q=torch.zeros(2, 3, 4, 258), k=torch.zeros(2, 3, 2, 258)),
        dict(q=q.transpose(2, 3).contiguous().transpose(2, 3)), dict(q_weight=w[:32]), dict(q_weight=w.double()), dict(q_weight=w.bfloat16()),
        dict(q_weight=torch.ones(128)[::2]), dict(q=q.bfloat16(), k=k.bfloat16(), q_weight=w, k_weight=w.bfloat16()),
        dict(rotary=table.double()), dict(rotary=table[:, :63]), dict(rotary=rotary_table(8, 66)), dict(rotary=table[:2]),
        dict(rotary=table.clone().requires_grad_(True)), dict(positions=torch.zeros(3, dtype=torch.int32)),
        dict(rotary=table, positions=torch.zeros(3)), dict(rotary=table, positions=torch.zeros(4, dtype=torch.int32)),
        dict(rotary=table, positions=torch.zeros(1, 3, dtype=torch.int32)), dict(rotary=table, positions=torch.zeros(6, dtype=torch.int32)[::2]),
        dict(rotary=table.to("meta")),
    ):
        with pytest.raises(ValueError):
            qk_norm_rotary(**{"q": q, "k": k, **bad})
    for bad in ((-1, 4), (4, 3), (4, 4, 0.0)):
        with pytest.raises(ValueError):
            rotary_table(*bad)


def test_rotary_table_at_far_positions():
    t = rotary_table(100001, 8, base=10000.0)
    import math
    for p in (0, 1, 4097, 100000):
        for i in range(4):
            a = p * 10000.0 ** (-2 * i / 8)
            assert abs(t[p, i].item() - math.cos(a)) <= 2.0 ** -24 and abs(t[p, 4 + i].item() - math.sin(a)) <= 2.0 ** -24


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(monkeypatch, grad):
    """No operand requires grad, so nothing is recorded; a tangent must not vanish all the same."""
    from torch.autograd import forward_ad as fw

    from mmlearn_amd import attention as A

    monkeypatch.setattr(A.K, "require_gpu", lambda *a: None)
    monkeypatch.setattr(A.K, "qk_norm_rotary_fwd", lambda q, k, *a: (torch.empty(q.shape), torch.empty(k.shape)))
    ops = [torch.zeros(1, 2, 3, 4), torch.zeros(1, 2, 1, 4), torch.ones(4), torch.ones(4)]
    with torch.set_grad_enabled(grad), fw.dual_level():
        assert qk_norm_rotary(*ops)[0].shape == (1, 2, 3, 4)       # nothing has a tangent
        for n in range(4):
            duals = [fw.make_dual(t, torch.ones_like(t)) if i == n else t for i, t in enumerate(ops)]
            with pytest.raises((NotImplementedError, RuntimeError), match="forward|jvp"):
                qk_norm_rotary(*duals)
    with pytest.raises((NotImplementedError, RuntimeError), match="forward|jvp"):
        torch.func.jvp(lambda x: qk_norm_rotary(x, x)[0], (ops[0],), (ops[0],))
