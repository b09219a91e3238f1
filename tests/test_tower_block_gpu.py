"""The tower operators as they run together: packed projection -> per-head norm and rotation of queries and keys -> attention with the
learned relative bias -> output projection, its gradients in float64, the optimizer step on them, and the same block token by token."""

import math

import pytest
import torch
import torch.nn.functional as F

from mmlearn_amd.attention import qk_norm_rotary, relative_attention, rotary_table
from mmlearn_amd.optim import AdamW, Muon
from oracle import tower_oracle as oracle

B, L, E, H, HK, D = 3, 90, 192, 4, 2, 64


class Block(torch.nn.Module):
    """f32 parameters, bf16 arithmetic, as under autocast."""

    def __init__(self):
        super().__init__()
        g = torch.Generator().manual_seed(11)
        self.qkv = torch.nn.Parameter(torch.randn((H + 2 * HK) * D, E, generator=g) / math.sqrt(E))
        self.proj = torch.nn.Parameter(torch.randn(E, H * D, generator=g) / math.sqrt(H * D))
        self.qw = torch.nn.Parameter(1 + 0.2 * torch.randn(D, generator=g))
        self.kw = torch.nn.Parameter(1 + 0.2 * torch.randn(D, generator=g))
        self.bias = torch.nn.Parameter(torch.randn(16, H, generator=g))
        self.register_buffer("rotary", rotary_table(L, 32))

    def heads(self, x, positions=None):
        y = F.linear(x, self.qkv.to(x.dtype)).view(*x.shape[:2], H + 2 * HK, D)
        q, k = qk_norm_rotary(y[:, :, :H], y[:, :, H:H + HK], self.qw, self.kw, rotary=self.rotary, positions=positions)
        return q.transpose(1, 2), k.transpose(1, 2), y[:, :, H + HK:].transpose(1, 2)

    def forward(self, x, mask=None):
        q, k, v = self.heads(x)
        o = relative_attention(q, k, v, self.bias, max_distance=40, bidirectional=False, causal=True, key_mask=mask)
        return F.linear(o.flatten(2), self.proj.to(x.dtype))


def _oracle(block, x, keep):
    p = {n: t.detach().double().cpu().requires_grad_(True) for n, t in block.named_parameters()}
    x = x.double().cpu().requires_grad_(True)
    y = (x @ p["qkv"].T).view(B, L, H + 2 * HK, D)
    t = block.rotary.double().cpu()
    q = oracle.qk_norm_rotary(y[:, :, :H], p["qw"], t, None, False, 1e-6).transpose(1, 2)
    k = oracle.qk_norm_rotary(y[:, :, H:H + HK], p["kw"], t, None, False, 1e-6).transpose(1, 2)
    o = oracle.relative_attention(q, k, y[:, :, H + HK:].transpose(1, 2), p["bias"], 40, False, None, True, keep)
    return o.flatten(2) @ p["proj"].T, p, x


def _inputs():
    g = torch.Generator().manual_seed(12)
    x, dy = (torch.randn(B, L, E, generator=g).bfloat16().cuda() for _ in range(2))
    lengths = torch.tensor([L, 37, 0], dtype=torch.int32)
    return x, dy, lengths, torch.arange(L)[None] < lengths[:, None]


@pytest.mark.gpu
def test_block_and_step():
    block = Block().cuda()
    x, dy, lengths, keep = _inputs()
    x.requires_grad_(True)
    y = block(x, lengths.cuda())
    y.backward(dy)
    want, p, xd = _oracle(block, x.detach(), keep)
    names = list(p)
    grads = dict(zip([*names, "x"], torch.autograd.grad(want, [*p.values(), xd], dy.double().cpu())))
    # a value passes at most 16 roundings to bf16 on its way (weights, projections, norm, P, o, dS, the gradients of each), each off by half a
    # step at most and by 2^-9 in the mean square
    tol = 16 * 2.0 ** -9
    assert (y.detach().double().cpu() - want).norm() <= tol * want.norm()
    for n, t in [*block.named_parameters(), ("x", x)]:
        assert (t.grad.double().cpu() - grads[n]).norm() <= tol * grads[n].norm(), n

    matrices, rest = [block.qkv, block.proj], [block.qw, block.kw, block.bias]
    before = [t.detach().double().cpu() for t in matrices]
    kept = [t.detach().clone() for t in rest]
    Muon(matrices, lr=0.05, weight_decay=0.0).step()
    AdamW(rest, lr=1e-3).step()
    for w, old in zip(matrices, before):
        g = 1.95 * w.grad.double().cpu()      # first step: g + 0.95 g
        o = oracle.orthogonalize(g)
        moved = (w.detach().double().cpu() - old) / (-0.05 * math.sqrt(max(1.0, w.shape[0] / w.shape[1])))
        assert (moved - o).norm() <= 1e-2 * o.norm()
    assert all(not torch.equal(t.detach(), k) for t, k in zip(rest, kept))


@pytest.mark.gpu
def test_token_by_token_gives_the_whole_sequence():
    block = Block().cuda().requires_grad_(False)
    x, _, _, _ = _inputs()
    whole = block(x)
    keys = torch.zeros(B, L, HK, D, dtype=torch.bfloat16, device="cuda")
    values = torch.full_like(keys, float("nan"))     # nobody has written there yet
    for i in range(L):
        at = torch.full((1,), i, dtype=torch.int64, device="cuda")
        q, k, v = block.heads(x[:, i:i + 1], at)
        keys[:, i], values[:, i] = k[:, :, 0], v[:, :, 0]
        n = torch.full((B,), i + 1, dtype=torch.int32, device="cuda")
        o = relative_attention(q, keys.transpose(1, 2), values.transpose(1, 2), block.bias, max_distance=40, bidirectional=False, causal=True,
                               key_mask=n, q_offset=n - 1)
        y = F.linear(o.flatten(2), block.proj.bfloat16())
        # the same roundings but for the order of sums, which may turn a rounding of P, of o and of y the other way
        assert (y[:, 0].double() - whole[:, i].double()).norm() <= 4 * 2.0 ** -8 * whole[:, i].double().norm(), i


@pytest.mark.gpu
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_training_step_is_the_eager_one(backend):
    """``torch.compile`` breaks its graph around the operators and the optimizer's step and computes what the eager step does."""
    x, dy, lengths, _ = _inputs()
    lengths = lengths.cuda()

    def step(block, opt):
        y = block(x, lengths)
        y.backward(dy)
        opt.step()
        opt.zero_grad()
        return y.detach()

    torch._dynamo.reset()
    results = []
    for compiled in (False, True):
        block = Block().cuda()
        opt = Muon([block.qkv, block.proj], lr=0.05)
        run = torch.compile(step, backend=backend) if compiled else step
        results.append([run(block, opt) for _ in range(3)] + [block.qkv.detach(), block.proj.detach(), block.bias.grad])
    for a, b in zip(*results):
        assert (a is None and b is None) or torch.equal(a, b)
    held = torch.randn(40, 50, device="cuda")
    from mmlearn_amd.optim import orthogonalize

    assert torch.equal(torch.compile(lambda t: orthogonalize(2 * t), backend=backend)(held), orthogonalize(2 * held))
    torch._dynamo.reset()
