"""Attention with a learned relative position bias against its float64 definition: lengths, head layouts, types, bucket schemes, masks with
anything behind them, offsets, strides; gradients (table included) against the definition's and against differences; refusals."""

import ctypes
import math
import os
import subprocess

import pytest
import torch

from mmlearn_amd import kernels as K
from mmlearn_amd.attention import relative_attention
from oracle import tower_oracle as oracle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _case(B, H, Hk, Lq, Lk, D, dtype="bfloat16", table="same", buckets=32, far=128, bidir=True, causal=False, mask=None, offset=0, strides="rows"):
    return dict(B=B, H=H, Hk=Hk, Lq=Lq, Lk=Lk, D=D, dtype=dtype, table=table, buckets=buckets, far=far, bidir=bidir, causal=causal, mask=mask,
                offset=offset, strides=strides)


CASES = [
    # one token
    _case(1, 1, 1, 1, 1, 64),
    _case(2, 4, 4, 1, 333, 64, causal=True, bidir=False, offset=332),
    _case(3, 8, 2, 1, 700, 128, mask="lengths", causal=True, bidir=False, offset="tensor"),
    _case(2, 6, 1, 5, 129, 128, "float16", mask="bool", offset=40),
    _case(2, 32, 1, 1, 65, 64, mask="int64"),
    _case(1, 2, 2, 3, 3000, 64, "float16", far=40, buckets=16, offset=2997),
    _case(2, 3, 3, 4, 31, 128, mask="len64", offset=-7, causal=True),
    _case(1, 40, 1, 1, 100, 64),                     # 40 query heads on one key head: more rows than the few-rows kernel holds
    _case(1, 32, 1, 1, 90, 128, far=512, buckets=64),   # bias vectors of 32 heads that its LDS cannot hold
    # whole sequences
    _case(2, 3, 3, 33, 33, 64),
    _case(2, 4, 2, 64, 64, 64, causal=True),
    _case(1, 2, 1, 65, 63, 128, "float16", "f32", bidir=False),
    _case(2, 3, 1, 77, 77, 64, "float16", "f32", mask="lengths", strides="heads"),
    _case(2, 2, 2, 129, 200, 128, mask="bool", strides="packed"),
    _case(2, 4, 1, 300, 300, 64, "bfloat16", "f32", buckets=16, far=20, causal=True, bidir=False),
    _case(1, 2, 2, 257, 513, 64, buckets=8, far=9, mask="uint8", offset=200),
    _case(1, 2, 1, 150, 513, 128, buckets=8, far=17, causal=True, offset=363, mask="int32"),
    _case(1, 2, 2, 513, 100, 128, "float16", buckets=4, far=2, offset=-300),
    _case(2, 2, 1, 200, 140, 64, causal=True, offset=-60, mask="lengths", bidir=False),   # early rows see no key
    _case(1, 1, 1, 130, 700, 64, buckets=256, far=512, offset=300),
    _case(1, 2, 2, 70, 70, 64, buckets=2, far=1, bidir=False),
    _case(1, 2, 2, 40, 40, 64, offset=1 << 28),
    _case(5, 2, 2, 48, 48, 64, mask="tensor of none"),
    # more heads than go together on an XCD, and a few left over
    _case(3, 25, 5, 130, 130, 64, causal=True),
    _case(2, 38, 38, 40, 70, 128, "float16", mask="lengths"),
]


def _layout(x, kind):
    if kind == "rows":      # [B, L, H, D] behind [B, H, L, D]
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if kind == "packed":    # rows of a wider projection
        B, H, L, D = x.shape
        wide = torch.full((B, L, H + 2, D), float("nan"), dtype=x.dtype, device=x.device)
        wide[:, :, 1:1 + H] = x.transpose(1, 2)
        return wide[:, :, 1:1 + H].transpose(1, 2)
    return x.contiguous()


def _inputs(c, seed=0, spoil=True):
    g = torch.Generator().manual_seed(seed)
    dt = getattr(torch, c["dtype"])
    B, H, Hk, Lq, Lk, D = (c[n] for n in ("B", "H", "Hk", "Lq", "Lk", "D"))
    q = torch.randn(B, H, Lq, D, generator=g).to(dt)
    k, v = (torch.randn(B, Hk, Lk, D, generator=g).to(dt) for _ in range(2))
    table = torch.randn(c["buckets"], H, generator=g).to(torch.float32 if c["table"] == "f32" else dt)
    dout = torch.randn(B, Lq, H, D, generator=g).to(dt)
    keep, mask = None, None
    if c["mask"] in ("lengths", "len64"):
        n = torch.randint(0, Lk + 1, (B,), generator=g)
        n[0], n[-1] = Lk, 0
        keep = torch.arange(Lk)[None] < n[:, None]
        mask = n.to(torch.int32 if c["mask"] == "lengths" else torch.int64)
        mask = mask if c["mask"] == "lengths" else mask * 3 - 2 * n   # (the same numbers)
    elif c["mask"] == "tensor of none":
        keep = torch.ones(B, Lk, dtype=torch.bool)
        keep[1] = False
        keep[2, 1:] = False
        keep[3, :-1] = False
        mask = keep
    elif c["mask"]:
        keep = torch.rand(B, Lk, generator=g) < 0.6
        keep[0, 64:128] = False    # a tile that holds nothing
        if B > 1:
            keep[-1] = False       # a sample that holds nothing
        mask = {"bool": keep, "uint8": keep.to(torch.uint8) * 3, "int32": keep.int() * -5, "int64": keep.long() << 40}[c["mask"]]
        wide = torch.ones(B, Lk + 7, dtype=mask.dtype)
        wide[:, :Lk] = mask
        mask = wide[:, :Lk]
    if keep is not None and spoil:   # what masked keys hold does not matter
        bad = (~keep)[:, None, :, None]
        k = torch.where(bad, torch.tensor(float("nan")), k.float()).to(dt)
        v = torch.where(bad, torch.tensor(float("inf")), v.float()).to(dt)
    offset = c["offset"]
    if offset == "tensor":
        offset = (keep.sum(1) - 1 if keep is not None else torch.arange(B)).int()
    dev = [_layout(t.cuda(), c["strides"]) for t in (q, k, v)] + [table.cuda(), dout.cuda()]
    if isinstance(mask, torch.Tensor):
        cuda_mask = mask.cuda()
        if mask.dim() == 2:
            full = torch.ones(B, Lk + 7, dtype=mask.dtype, device="cuda")
            full[:, :Lk] = cuda_mask
            cuda_mask = full[:, :Lk]
        mask = cuda_mask
    return dev, mask, keep, offset


def _bounds(c, q, k, v, table, dout, keep, offset):
    """Float64 results and, beside each, how far the kernels' roundings may carry them: half a step of the operands' type for P, for dS and for
    every output; half a step of half a step for the P and the o that delta comes from, which are held in two parts; f32 for the rest."""
    dt = getattr(torch, c["dtype"])
    u = torch.finfo(dt).eps / 2
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0      # half a step of f16's smallest values
    B, H, Hk, Lq, Lk, D = (c[n] for n in ("B", "H", "Hk", "Lq", "Lk", "D"))
    G, scale = H // Hk, D ** -0.5
    out = {n: [] for n in ("out", "dq")}
    res = {n: torch.zeros(s, dtype=torch.float64) for n, s in (("out", (B, Lq, H, D)), ("dq", (B, H, Lq, D)), ("dk", (B, Hk, Lk, D)),
                                                                ("dv", (B, Hk, Lk, D)), ("dtable", (c["buckets"], H)))}
    err = {n: torch.zeros_like(t) for n, t in res.items()}
    keep = torch.ones(B, Lk, dtype=torch.bool) if keep is None else keep
    for b in range(B):
        off = offset if isinstance(offset, int) else int(offset[b])
        bm = oracle.bucket_map(Lq, Lk, off, c["buckets"], c["far"], c["bidir"])
        seen = keep[b][None].expand(Lq, Lk)
        if c["causal"]:
            seen = seen & (torch.arange(Lk)[None] <= torch.arange(Lq)[:, None] + off)
        for h in range(H):
            Q, Kb, Vb, dO = q[b, h], k[b, h // G] * keep[b][:, None], v[b, h // G] * keep[b][:, None], dout[b, :, h]
            Kb, Vb = (torch.where(keep[b][:, None], t[b, h // G], torch.zeros(())) for t in (k, v))
            bias = table[:, h][bm]
            z = (Q @ Kb.T) * scale + bias
            p = torch.where(seen, torch.exp(z - torch.where(seen, z, torch.full_like(z, -1e30)).amax(1, keepdim=True)), torch.zeros_like(z)) if Lk else z
            p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
            # a score: sums of D products, the scale, the bias, the maximum and the exponential, in f32; then the softmax's sum
            es = 2.0 ** -24 * ((D + 8) * ((Q.abs() @ Kb.abs().T) * scale).amax(1, keepdim=True) + 16 * bias.abs().max() + Lk / 16 + 32) if Lk else z
            A = p @ Vb.abs()
            eo = (u + es) * A + tiny * Vb.abs().sum(0) if Lk else torch.zeros(Lq, D, dtype=torch.float64)
            o = p @ Vb
            res["out"][b, :, h] = o
            err["out"][b, :, h] = u * o.abs() + eo + tiny
            if not Lk:
                continue
            dp = dO @ Vb.T
            delta = (dO * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            eo2 = (u * u + es) * A + tiny * Vb.abs().sum(0)
            edelta = (dO.abs() * (u * u * o.abs() + eo2 + tiny)).sum(1, keepdim=True)
            f32 = p * 2.0 ** -24 * (D + 8) * (dO.abs() @ Vb.abs().T + (dO.abs() * o.abs()).sum(1, keepdim=True))
            e32 = 2 * es * ds.abs() + p * edelta + f32           # dS before its rounding
            e16 = e32 + u * ds.abs() + tiny
            res["dq"][b, h] = ds @ Kb * scale
            err["dq"][b, h] = e16 @ Kb.abs() * scale
            res["dk"][b, h // G] += ds.T @ Q * scale
            err["dk"][b, h // G] += e16.T @ Q.abs() * scale
            res["dv"][b, h // G] += p.T @ dO
            err["dv"][b, h // G] += ((u + 2 * es) * p + tiny).T @ dO.abs()
            res["dtable"][:, h].index_add_(0, bm.reshape(-1), ds.reshape(-1))
            err["dtable"][:, h].index_add_(0, bm.reshape(-1), (e32 + 2.0 ** -24 * 64 * ds.abs()).reshape(-1))
    ut = torch.finfo(torch.float32 if c["table"] == "f32" else dt).eps / 2
    for n in ("dq", "dk", "dv", "dtable"):
        w = ut if n == "dtable" else u
        err[n] = err[n] * 1.01 + w * res[n].abs() + (tiny if w == u else 0.0) + 2.0 ** -24 * 32 * res[n].abs().max() if res[n].numel() else err[n]
    return res, err


def _run(c, dev, mask, offset):
    leaves = [t.detach().requires_grad_(True) for t in dev[:4]]
    off = offset.cuda() if isinstance(offset, torch.Tensor) else offset
    out = relative_attention(*leaves, max_distance=c["far"], bidirectional=c["bidir"], causal=c["causal"], key_mask=mask, q_offset=off)
    grads = torch.autograd.grad(out, leaves, dev[4])
    return dict(zip(("out", "dq", "dk", "dv", "dtable"), [t.detach() for t in (out, *grads)]))


@pytest.mark.gpu
@pytest.mark.parametrize("c", CASES, ids=lambda c: "-".join(str(v) for v in c.values()))
def test_against_float64(c):
    dev, mask, keep, offset = _inputs(c)
    got = _run(c, dev, mask, offset)
    res, err = _bounds(c, *(t.double().cpu() for t in dev), keep, offset)
    assert got["out"].is_contiguous()
    for n in res:
        x = got[n].double().cpu()
        assert x.shape == res[n].shape and torch.isfinite(x).all(), n
        over = ((x - res[n]).abs() - err[n] * 1.01).max().item() if x.numel() else 0.0
        assert over <= 0, (n, over, (x - res[n]).norm().item() / max(res[n].norm().item(), 1e-300))
        # the bounds are sums of absolute values: also hold the whole to what independent roundings leave of them
        if res[n].norm() > 0 and n != "dtable":
            assert (x - res[n]).norm() <= 6 * torch.finfo(dev[0].dtype).eps * res[n].norm(), n
    with torch.no_grad():
        off = offset.cuda() if isinstance(offset, torch.Tensor) else offset
        again = relative_attention(*dev[:4], max_distance=c["far"], bidirectional=c["bidir"], causal=c["causal"], key_mask=mask, q_offset=off)
    # (a pass that records sums P in two parts: the same value, rounded elsewhere)
    assert again.shape == got["out"].shape and ((again.double().cpu() - res["out"]).abs() <= err["out"] * 1.01).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype,lq", [(64, "bfloat16", 300), (128, "bfloat16", 300), (64, "float16", 300), (128, "bfloat16", 3)])
def test_table_gradient_in_f32(D, dtype, lq):
    """An f32 table's gradient is no 16-bit one.  What 16 bits do to it goes through delta: with P and o rounded once (u = 2^-8 in bf16) it is
    off by about u of its size, 4e-3; in two parts each, by about u^2 = 1.5e-5.  The scores' f32 sums add about 128 * 2^-24 = 8e-6."""
    c = _case(2, 2, 1, lq, 300, D, dtype, "f32", buckets=16, far=64, mask="bool", offset=40)
    dev, mask, keep, offset = _inputs(c, 6)
    got = _run(c, dev, mask, offset)
    res, err = _bounds(c, *(t.double().cpu() for t in dev), keep, offset)
    assert got["dtable"].dtype == torch.float32
    off = (got["dtable"].double().cpu() - res["dtable"]).norm() / res["dtable"].norm()
    assert off <= 2e-4, off.item()


@pytest.mark.gpu
def test_gradients_against_differences():
    c = _case(2, 2, 1, 37, 45, 64, "float16", "f32", buckets=8, far=12, mask="bool", offset=3)
    dev, mask, keep, offset = _inputs(c, 4)
    got = _run(c, dev, mask, offset)
    g = torch.Generator().manual_seed(2)
    a = [torch.where(torch.isfinite(t), t, torch.zeros((), dtype=t.dtype, device=t.device)).double().cpu() for t in dev]
    for n, name in enumerate(("dq", "dk", "dv", "dtable")):
        d = torch.randn(a[n].shape, generator=g, dtype=torch.float64)
        f = []
        for t in (1e-4, -1e-4):
            x = list(a[:4])
            x[n] = x[n] + t * d
            f.append((oracle.relative_attention(*x, max_distance=12, keep=keep, q_offset=offset) * a[4]).sum().item())
        want = (f[0] - f[1]) / 2e-4
        # every element of the gradient carries a few half steps of f16, independent of the direction's signs
        tol = 8 * torch.finfo(torch.float16).eps * (got[name].double().cpu() * d).norm().item() * 4 + 1e-5 * abs(want)
        assert abs((got[name].double().cpu() * d).sum().item() - want) <= tol + 2.0 ** -24 * d.numel(), name


@pytest.mark.gpu
def test_infinite_table_entries_forbid_a_bucket():
    c = _case(1, 2, 2, 70, 70, 64, "bfloat16", "f32", buckets=8, far=12)
    dev, mask, keep, offset = _inputs(c, 6)
    dev[3][4:] = float("-inf")     # nothing behind the query
    dev[3][0, 1] = float("-inf")   # nor itself, for head 1: row 0 keeps no key
    got = _run(c, dev, mask, offset)
    q, k, v, t, do = (x.double().cpu() for x in dev)
    rel = torch.arange(70)[None] - torch.arange(70)[:, None]
    b = oracle.bucket_map(70, 70, 0, 8, 12, True)
    z = (q @ k.transpose(2, 3)) / 8 + t[b].permute(2, 0, 1)
    p = torch.nan_to_num(torch.softmax(z, -1), nan=0.0)
    want = (p @ v).transpose(1, 2)
    assert not got["out"][0, 0, 1].any() and all(torch.isfinite(x).all() for x in got.values())
    assert (got["out"].double().cpu() - want).norm() <= 6 * 2.0 ** -8 * want.norm()
    assert not got["dtable"][4:].any() and got["dtable"][0, 1] == 0


@pytest.mark.gpu
def test_no_rows_no_keys_no_samples():
    table = torch.randn(32, 2, device="cuda", requires_grad=True)
    for B, Lq, Lk in ((2, 0, 5), (2, 5, 0), (0, 4, 4), (1, 200, 0), (2, 0, 0)):
        q = torch.randn(B, 2, Lq, 64, device="cuda").bfloat16().requires_grad_(True)
        k, v = (torch.randn(B, 2, Lk, 64, device="cuda").bfloat16().requires_grad_(True) for _ in range(2))
        out = relative_attention(q, k, v, table)
        grads = torch.autograd.grad(out, (q, k, v, table), torch.ones_like(out))
        assert out.shape == (B, Lq, 2, 64) and not out.any() and all(not g.any() and g.shape == t.shape for g, t in zip(grads, (q, k, v, table)))


@pytest.mark.gpu
@pytest.mark.parametrize("B,lk,shape,dtype", [(0, 9, (0, 9), torch.bool), (0, 9, (0,), torch.int32), (3, 0, (3, 0), torch.int64), (3, 0, (3,), torch.int64)])
def test_masks_of_nothing(B, lk, shape, dtype):
    q, k = (torch.randn(B, n, 2, 64, device="cuda").bfloat16().transpose(1, 2).requires_grad_() for n in (5, lk))
    table = torch.randn(8, 2, device="cuda", requires_grad=True)
    off = torch.zeros(B, dtype=torch.int32, device="cuda")
    out = relative_attention(q, k, k, table, key_mask=torch.zeros(shape, dtype=dtype, device="cuda"), q_offset=off)
    assert out.shape == (B, 5, 2, 64) and not out.any()
    for g, t in zip(torch.autograd.grad(out, (q, k, table), torch.ones_like(out)), (q, k, table)):
        assert g.shape == t.shape and not g.any()


@pytest.mark.gpu
def test_rows_more_than_32_bits_apart():
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 22 GiB of device memory")
    g = torch.Generator().manual_seed(8)
    L, far = 620, 1 << 23
    store = torch.empty(L * far, dtype=torch.bfloat16, device="cuda")     # the last rows lie past 2^32 elements
    rows = torch.randn(2, 1, 1, L, 64, generator=g).bfloat16().cuda()
    k, v = (store.as_strided((1, 1, L, 64), (0, 0, far, 1), o) for o in (0, 64))
    k.copy_(rows[0])
    v.copy_(rows[1])
    q = torch.randn(1, 1, 200, 64, generator=g).bfloat16().cuda()
    table = torch.randn(32, 1, generator=g).cuda()
    for n in (1, 200):
        a = relative_attention(q[:, :, :n], k, v, table, q_offset=400)
        assert torch.equal(a, relative_attention(q[:, :, :n], rows[0], rows[1], table, q_offset=400))


@pytest.mark.gpu
def test_repeatable_captured_and_on_two_streams():
    cs = [_case(4, 8, 2, 130, 130, 64, mask="bool"), _case(4, 8, 2, 1, 900, 64, causal=True, bidir=False, mask="lengths", offset="tensor")]
    for c in cs:
        dev, mask, keep, offset = _inputs(c)
        want = {n: t.clone() for n, t in _run(c, dev, mask, offset).items()}
        offset = offset.cuda() if isinstance(offset, torch.Tensor) else offset
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        got = []
        for s in (s1, s2, s1):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(_run(c, dev, mask, offset))
        for s in (s1, s2):
            torch.cuda.current_stream().wait_stream(s)
        for other in got:
            assert all(torch.equal(other[n], want[n]) for n in want)
        graphs = []
        torch.cuda.synchronize()
        for _ in range(2):     # two graphs: each has workspaces of its own
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                held = _run(c, dev, mask, offset)
            graphs.append((graph, held))
        for _ in range(3):
            for graph, held in graphs:
                for t in held.values():
                    t.fill_(3.0)
                graph.replay()
            torch.cuda.synchronize()
            for graph, held in graphs:
                assert all(torch.equal(held[n], want[n]) for n in want)
            fresh = _run(c, dev, mask, offset)
            assert all(torch.equal(fresh[n], want[n]) for n in want)


@pytest.mark.gpu
def test_only_some_gradients_are_wanted():
    c = _case(2, 2, 1, 66, 66, 64)
    dev, mask, keep, offset = _inputs(c)
    want = _run(c, dev, mask, offset)
    for n, name in enumerate(("dq", "dk", "dv", "dtable")):
        leaves = [t.detach() for t in dev[:4]]
        leaves[n].requires_grad_(True)
        out = relative_attention(*leaves)
        (got,) = torch.autograd.grad(out, leaves[n], dev[4].expand(2, *dev[4].shape[1:]))
        assert torch.equal(got, want[name]), name


def test_struct_layout_matches_header():
    from mmlearn_amd import _lib

    src = '#include <stdio.h>\n#include "mmlearn_hip.h"\nint main(){printf("%zu %zu", sizeof(mmk_rel_attn), offsetof(mmk_rel_attn, scale));return 0;}'
    exe = "/tmp/_mmk_rel_sizeof"
    subprocess.run(["gcc", "-x", "c", "-", "-I", os.path.join(ROOT, "include"), "-o", exe], input=src, text=True, check=True)
    size, scale = map(int, subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split())
    assert ctypes.sizeof(_lib.RelAttn) == size and _lib.RelAttn.scale.offset == scale


def test_bucket_borders():
    for buckets, far, bidir in ((32, 128, True), (32, 128, False), (64, 256, True), (16, 40, True), (2, 1, False), (4, 2, True), (256, 512, True), (8, 9, True)):
        near, borders, n = K.relative_buckets(buckets, far, bidir)
        side = buckets // 2 if bidir else buckets
        assert near == side // 2 and n == side - near - 1
        for d in range(far + 5):
            mine = d if d < near else near + sum(min(d, far) >= borders[t] for t in range(n))
            assert mine == oracle.bucket(-min(d, far), buckets, far, bidir), (buckets, far, bidir, d)


def test_buckets_agree_with_the_hf_text_models():
    modeling = pytest.importorskip("transformers.models.t5.modeling_t5")
    rel = torch.arange(-300, 301)
    for bidir in (True, False):
        want = modeling.T5Attention._relative_position_bucket(rel, bidir, 32, 128)
        assert want.tolist() == [oracle.bucket(max(-128, min(128, r)), 32, 128, bidir) for r in rel.tolist()]


def test_refusals(monkeypatch):
    from mmlearn_amd import attention as A

    def bf(*shape):
        return torch.zeros(*shape, dtype=torch.bfloat16)

    with pytest.raises(RuntimeError, match="no CPU fallback"):
        relative_attention(bf(1, 1, 1, 64), bf(1, 1, 1, 64), bf(1, 1, 1, 64), torch.zeros(32, 1))
    monkeypatch.setattr(A.K, "require_gpu", lambda *a: None)
    monkeypatch.setattr(A._RelativeAttention, "apply", lambda *a: pytest.fail("reached the kernel"))
    q, k, t = bf(2, 4, 6, 64), bf(2, 2, 8, 64), torch.zeros(32, 4)
    flat = bf(2 * 4 * 6 * 64 + 8)
    for bad in (
        dict(q=q[0]), dict(q=q.float(), k=k.float(), v=k.float()), dict(k=k.half()), dict(v=k[:, :, :7]), dict(k=k[:1], v=k[:1]), dict(k=bf(2, 3, 8, 64), v=bf(2, 3, 8, 64)),
        dict(q=bf(2, 4, 6, 32), k=bf(2, 2, 8, 32), v=bf(2, 2, 8, 32)), dict(k=bf(2, 0, 8, 64), v=bf(2, 0, 8, 64)), dict(q=bf(2, 4, 6, 128)[..., ::2]),
        dict(q=bf(2, 4, 6, 68)[..., :64]), dict(q=flat[1:1 + q.numel()].view(q.shape)), dict(table=t[:, :3]), dict(table=t.bfloat16().half()), dict(table=t[0]),
        dict(table=torch.zeros(4, 32).t()), dict(table=torch.zeros(31, 4)), dict(table=torch.zeros(2, 4)), dict(table=torch.zeros(258, 4)),
        dict(table=torch.zeros(1, 4), bidirectional=False), dict(max_distance=8), dict(max_distance=513), dict(max_distance=16.5),
        dict(key_mask=torch.ones(2, 7, dtype=torch.bool)), dict(key_mask=torch.ones(2, 8)), dict(key_mask=torch.ones(2, 8, dtype=torch.int16)), dict(key_mask=torch.ones(3, dtype=torch.int32)),
        dict(key_mask=torch.ones(2, dtype=torch.bool)), dict(key_mask=torch.ones(8, 2, dtype=torch.bool).t()), dict(key_mask=torch.ones(1, 8, dtype=torch.bool)),
        dict(q_offset=1.5), dict(q_offset=1 << 29), dict(q_offset=torch.zeros(2)), dict(q_offset=torch.zeros(3, dtype=torch.int32)), dict(q_offset=torch.zeros(2, dtype=torch.int64)),
        dict(table=t.to("meta")),
    ):
        with pytest.raises(ValueError):
            relative_attention(**{"q": q, "k": k, "v": k, "table": t, **bad})


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(monkeypatch, grad):
    """No operand requires grad, so nothing is recorded; a tangent must not vanish all the same."""
    from torch.autograd import forward_ad as fw

    from mmlearn_amd import attention as A

    monkeypatch.setattr(A.K, "require_gpu", lambda *a: None)
    monkeypatch.setattr(A.K, "rel_attn_operands", lambda *a: None)
    monkeypatch.setattr(A.K, "rel_attn_fwd", lambda p, q, record: (q.transpose(1, 2).contiguous(), None, None))
    ops = [torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16) for _ in range(3)] + [torch.zeros(32, 2)]
    with torch.set_grad_enabled(grad), fw.dual_level():
        assert relative_attention(*ops).shape == (1, 3, 2, 64)     # nothing has a tangent
        for n in range(4):
            duals = [fw.make_dual(t, torch.ones_like(t)) if i == n else t for i, t in enumerate(ops)]
            with pytest.raises((NotImplementedError, RuntimeError), match="forward|jvp"):
                relative_attention(*duals)


def _exact_head(q, k, v, dout, scale, seen=None):
    """One head without bias in float64: out, dq, dk, dv, and dS, P."""
    z = (q @ k.T) * scale
    if seen is not None:
        z = z.masked_fill(~seen, float("-inf"))
    p = torch.softmax(z, 1)
    o = p @ v
    ds = p * (dout @ v.T - (dout * o).sum(1, keepdim=True))
    return o, ds @ k * scale, ds.T @ q * scale, p.T @ dout, ds, p


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lq,lk,size,peak", [(64, 4096, 1e-4, 1.0), (300, 512, 1e-5, 1.0), (96, 96, 1e4, 3.0), (1, 4096, 1e-4, 1.0), (40, 700, 1e4, 3.0),
                                             (1100, 300, 1e-4, 1.0)])     # (several workgroups a key block)
def test_f16_gradients_of_any_size(lq, lk, size, peak, D):
    """dS = P (dP - delta) stays off both ends of f16's range, whatever the size of the gradient that comes in: it is rounded once relative to its
    size, as the results are.  (Rounded as it stands it is subnormal at ordinary sizes of P and dout, and infinite beyond 65504.)"""
    g = torch.Generator().manual_seed(lq + lk)
    q = (peak * torch.randn(1, 1, lq, D, generator=g)).half()
    k, v = (torch.randn(1, 1, lk, D, generator=g).half() for _ in range(2))
    dout = (size * torch.randn(1, lq, 1, D, generator=g)).clamp(-6e4, 6e4).half()
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v, torch.zeros(32, 1))]
    out = relative_attention(*leaves)
    got = [t.double().cpu() for t in torch.autograd.grad(out, leaves, dout.cuda())]
    Q, Kd, V, dO = q[0, 0].double(), k[0, 0].double(), v[0, 0].double(), dout[0, :, 0].double()
    scale = D ** -0.5
    o, dq, dk, dv, ds, p = _exact_head(Q, Kd, V, dO, scale)
    u = 2.0 ** -11
    # a score's f32 sums (D products, scale, maximum, exponential, softmax's sum), as a relative error of P; delta from an o in two parts of f16
    es = 2.0 ** -24 * ((D + 8) * (Q.abs() @ Kd.abs().T).amax(1, keepdim=True) * scale + lk / 16 + 32)
    edelta = (dO.abs() * (u * u * o.abs() + (u * u + es) * (p @ V.abs()) + 2.0 ** -25)).sum(1, keepdim=True)
    e32 = 2 * es * ds.abs() + p * edelta + p * 2.0 ** -24 * (D + 8) * (dO.abs() @ V.abs().T + (dO * o).abs().sum(1, keepdim=True))
    bounds = {"dq": ((u * ds.abs() + e32) @ Kd.abs() * scale, dq), "dk": ((u * ds.abs() + e32).T @ Q.abs() * scale, dk),
              "dv": (((u + 2 * es) * p).T @ dO.abs(), dv)}
    for (name, (err, want)), x in zip(bounds.items(), got):
        x = x[0, 0]
        fits = want.abs() < 6e4     # (a gradient of this size can itself be past f16's end, which is infinite and no fault)
        assert torch.isfinite(x[fits]).all() and fits.double().mean() > 0.99, name
        x = torch.where(fits, x, want)
        # the result is rounded once: half a step of its own size, or of f16's smallest values
        over = ((x - want).abs() - 1.01 * err - 1.01 * (u * want.abs() + 2.0 ** -25)).max().item()
        assert over <= 0, (name, over, ((x - want).norm() / want.norm()).item())
        # independent roundings: of dS (P) before the product, of the result after it
        once = (want.half().double() - want).norm()
        assert (x - want).norm() <= 2 * (once + u * want.norm()), (name, ((x - want).norm() / want.norm()).item())


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [1, 3, 130])
def test_f16_many_keys_far_below_the_first(lq):
    """2^20 keys, each 2^-26 of the first one's weight: together 1.5 % of the result, and none of them lost below f16's smallest values."""
    lk = 1 << 20
    far = 26 * math.log(2.0)
    q = torch.zeros(1, 1, lq, 64)
    q[..., 0] = 8.0                                       # scale 1 / 8: the score is k[0]
    k, v = torch.zeros(1, 1, lk, 64), torch.ones(1, 1, lk, 64)
    k[:, :, 0, 0], v[:, :, 0] = far, 0.0
    q, k, v = (t.half().cuda() for t in (q, k, v))
    weight = math.exp(-k[0, 0, 0, 0].double().item())     # of each of the others
    want = (lk - 1) * weight / (1 + (lk - 1) * weight)
    table = torch.zeros(32, 1, device="cuda")
    for grad in (False, True):
        out = relative_attention(q.requires_grad_(grad), k, v, table).double()
        # half a step of the result, and of P; the f32 sum of the weights: 2^14 tiles added to 1, each off by 2^-24 at most.  Times 2^7 a weight
        # is 32.2 times f16's smallest value 2^-24: each is off by half of that at most, 2^-25 / 2^7 of the largest one's weight
        assert (out - want).abs().max().item() <= want * (2 * 2.0 ** -11 + 2.0 ** -10) + lk * 2.0 ** -32, (grad, out.mean().item(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype", [(64, "bfloat16"), (128, "float16")])
@pytest.mark.parametrize("lq,used,tensor", [(1, 37, True), (3, 64, False), (1, 200, False), (70, 61, True), (200, 0, False)])
def test_causal_keys_behind_the_last_query_may_hold_anything(lq, used, tensor, D, dtype):
    """A cache of fixed size that nobody has filled beyond the newest token: causal alone keeps those places out."""
    g = torch.Generator().manual_seed(lq)
    lk, n = 300, used + lq
    dt = getattr(torch, dtype)
    q, k, v = (torch.randn(2, h, s, D, generator=g).to(dt).cuda() for h, s in ((4, lq), (2, n), (2, n)))
    dout = torch.randn(2, lq, 4, D, generator=g).to(dt).cuda()
    table = torch.randn(32, 4, generator=g).cuda()
    off = torch.full((2,), used, dtype=torch.int32, device="cuda") if tensor else used

    def run(k, v):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
        out = relative_attention(*leaves, causal=True, q_offset=off)
        with torch.no_grad():
            plain = relative_attention(*leaves, causal=True, q_offset=off)
        return out.detach(), plain, *torch.autograd.grad(out, leaves, dout)

    want = run(k, v)
    for junk in (float("nan"), float("inf")):
        big = [torch.full((2, 2, lk, D), junk, dtype=dt, device="cuda") for _ in range(2)]
        for b, t in zip(big, (k, v)):
            b[:, :, :n] = t
        got = run(*big)
        for name, a, b in zip(("out", "out without gradient", "dq", "dk", "dv", "dtable"), got, want):
            if name in ("dk", "dv"):
                assert not a[:, :, n:].any(), name     # (any() is true for a NaN)
                a = a[:, :, :n]
            # (another number of keys may divide the sums differently)
            assert torch.isfinite(a).all() and (a.double() - b.double()).norm() <= 4 * torch.finfo(dt).eps * b.double().norm(), name


def _described(B, H, Hk, Lq, Lk, D):
    """The C description of a call on operands that nobody reads."""
    from mmlearn_amd import _lib

    def flat(heads, rows):
        return torch.zeros(D, dtype=torch.bfloat16).as_strided((B, heads, rows, D), (0, 0, 0, 1))

    p = K.rel_attn_operands(flat(H, Lq), flat(Hk, Lk), flat(Hk, Lk), torch.zeros(32, H), 128, True, D ** -0.5, False, None, 0)
    return p, _lib.lib()


@pytest.mark.parametrize("B,H,Hk,Lq,Lk", [(64, 32, 1, 1, 1 << 20), (1, 2, 1, 130, 1 << 28), (1, 8, 8, 1, 1 << 28)])
def test_many_keys_are_not_many_rows(B, H, Hk, Lq, Lk):
    """What a launch holds is counted in queries; the length of a cache does not enter the forward's."""
    p, lib = _described(B, H, Hk, Lq, Lk, 64)
    assert lib.mmk_rel_attn_fwd_ws_floats(ctypes.byref(p)) >= 0, lib.mmk_last_error()
    assert (lib.mmk_rel_attn_bwd_ws_floats(ctypes.byref(p), 1) >= 0) == (B * Hk * Lk // 128 < 1 << 24)
    p, lib = _described(1 << 16, 1 << 8, 1, 1, 5, 64)     # 2^24 workgroups of 256 threads
    assert lib.mmk_rel_attn_fwd_ws_floats(ctypes.byref(p)) == -1 and b"query rows" in lib.mmk_last_error()


@pytest.mark.gpu
def test_a_batch_of_very_long_caches():
    """64 samples x 32 query heads against 2^20 keys (which all samples share here, by a stride of zero)."""
    g = torch.Generator().manual_seed(3)
    n = 1 << 20
    k, v = (torch.randn(1, 1, n, 64, generator=g).bfloat16().cuda() for _ in range(2))
    q = torch.randn(64, 32, 1, 64, generator=g).bfloat16().cuda()
    table = torch.randn(32, 32, generator=g).cuda()
    got = relative_attention(q, k.expand(64, -1, -1, -1), v.expand(64, -1, -1, -1), table, q_offset=n - 1)
    for b in (0, 40, 63):
        bias = torch.zeros(32, n, dtype=torch.float64, device="cuda") + table[15].double()[:, None]
        rel = oracle.bucket_map(1, 300, 299, 32, 128, True)[0].cuda()
        bias[:, -300:] = table.double()[rel].T
        p = torch.softmax((q[b, :, 0].double() @ k[0, 0].double().T) / 8 + bias, -1)
        want = p @ v[0, 0].double()
        # P and the result are each rounded once, with independent signs over the keys
        assert (got[b, 0].double() - want).norm() <= 2 * 2.0 ** -8 * want.norm(), b


@pytest.mark.gpu
def test_the_table_gradient_of_no_queries_needs_no_workspace():
    from mmlearn_amd import _lib

    q, kv = (torch.zeros(1, 2, n, 64, dtype=torch.bfloat16, device="cuda") for n in (0, 0))
    table, dtable = torch.zeros(32, 2, device="cuda"), torch.full((32, 2), 3.0, device="cuda")
    p, lib = K.rel_attn_operands(q, kv, kv, table, 128, True, 0.125, False, None, 0), _lib.lib()
    assert lib.mmk_rel_attn_bwd_ws_floats(ctypes.byref(p), 1) == 0
    _lib.check(lib.mmk_rel_attn_bwd(ctypes.byref(p), *[None] * 7, dtable.data_ptr(), None, _lib.stream()))
    assert not dtable.any()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1.0, 0.03, -0.2, 0.0])
@pytest.mark.parametrize("lq,dtype,train", [(1, "bfloat16", False), (150, "bfloat16", True), (70, "float16", True)])
def test_scales(lq, dtype, train, scale):
    """T5-type towers take scale = 1."""
    c = _case(2, 4, 2, lq, 190, 64, dtype, "f32")
    dev, _, _, _ = _inputs(c, 5)
    dev[0] = dev[0] / 4       # (scores of a few units at scale 1)
    leaves = [t.detach().requires_grad_(train) for t in dev[:4]]
    out = relative_attention(*leaves, scale=scale)
    a = [t.detach().double().cpu().requires_grad_(train) for t in dev[:4]]
    want = oracle.relative_attention(*a, scale=scale)
    # P, dS and the results are each rounded once, with independent signs: a few half steps of the type in the norm
    tol = 6 * torch.finfo(dev[0].dtype).eps
    assert (out.detach().double().cpu() - want.detach()).norm() <= tol * want.detach().norm()
    if train:
        got = torch.autograd.grad(out, leaves, dev[4])
        for name, x, w in zip(("dq", "dk", "dv", "dtable"), got, torch.autograd.grad(want, a, dev[4].double().cpu())):
            if scale == 0.0 and name in ("dq", "dk"):
                assert not x.any()
            else:
                assert (x.double().cpu() - w).norm() <= tol * w.norm(), name


@pytest.mark.gpu
@pytest.mark.parametrize("train", [False, True])
def test_a_serving_batch_with_offsets_of_its_own(train):
    """Each sample's new tokens stand behind its own cache: lengths and offsets a sample, a few tokens each."""
    g = torch.Generator().manual_seed(31)
    used = torch.tensor([0, 5, 63, 64, 250, 296], dtype=torch.int32)
    B, lq, lk = len(used), 4, 300
    q = torch.randn(B, lq, 8, 64, generator=g).bfloat16().cuda().transpose(1, 2)
    k, v = (torch.full((B, lk, 2, 64), float("nan"), dtype=torch.bfloat16) for _ in range(2))
    for b, n in enumerate((used + lq).tolist()):
        k[b, :n], v[b, :n] = (torch.randn(n, 2, 64, generator=g).bfloat16() for _ in range(2))
    table = torch.randn(32, 8, generator=g)
    keep = torch.arange(lk)[None] < (used + lq)[:, None]
    dout = torch.randn(B, lq, 8, 64, generator=g).bfloat16()
    leaves = [t.requires_grad_(train) for t in (q, k.cuda().transpose(1, 2), v.cuda().transpose(1, 2), table.cuda())]
    out = relative_attention(*leaves, bidirectional=False, causal=True, key_mask=(used + lq).cuda(), q_offset=used.cuda())
    a = [torch.nan_to_num(t.detach().double().cpu()).requires_grad_(train) for t in leaves]
    want = oracle.relative_attention(*a, bidirectional=False, causal=True, keep=keep, q_offset=used.tolist())
    tol = 6 * 2.0 ** -7
    assert (out.detach().double().cpu() - want.detach()).norm() <= tol * want.detach().norm()
    if train:
        for x, w in zip(torch.autograd.grad(out, leaves, dout.cuda()), torch.autograd.grad(want, a, dout.double())):
            assert torch.isfinite(x).all() and (x.double().cpu() - w).norm() <= tol * w.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("lq,lk,G", [(1, 1, 1), (1, 700, 4), (5, 3000, 6), (32, 90, 1)])
def test_few_rows_give_one_result_with_and_without_gradients(lq, lk, G, dtype):
    g = torch.Generator().manual_seed(lk)
    q, k, v = (torch.randn(2, h, n, 128, generator=g).to(getattr(torch, dtype)).cuda() for h, n in ((2 * G, lq), (2, lk), (2, lk)))
    table = torch.randn(32, 2 * G, generator=g).cuda()
    plain = relative_attention(q, k, v, table, q_offset=lk - lq)
    assert torch.equal(plain, relative_attention(q.requires_grad_(True), k, v, table, q_offset=lk - lq).detach())
    want = oracle.relative_attention(*(t.detach().double().cpu() for t in (q, k, v, table)), q_offset=lk - lq)
    # P in two parts is off by u^2: the result's one rounding (u at most, u / sqrt(3) in the mean square) is nearly all there is
    assert (plain.double().cpu() - want).norm() <= 0.75 * torch.finfo(q.dtype).eps / 2 * want.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("B,H,Hk,lq,lk,D,mask", [(3, 4, 2, 1, 1, 64, None), (2, 2, 1, 200, 1, 128, None), (4, 6, 3, 70, 40, 64, "one"), (2, 4, 4, 3, 500, 128, "one"),
                                                (1, 1, 1, 1200, 1, 64, None)])
def test_rows_with_one_key_pass_no_gradient_through_their_scores(B, H, Hk, lq, lk, D, mask, dtype):
    """A softmax over one key is 1 whatever its score: dq, dk and the table's gradient are zero, not small."""
    g = torch.Generator().manual_seed(lq + lk)
    dt = getattr(torch, dtype)
    q, k, v = (2 * torch.randn(B, h, n, D, generator=g).to(dt).cuda() for h, n in ((H, lq), (Hk, lk), (Hk, lk)))
    table, dout = torch.randn(32, H, generator=g).cuda(), torch.randn(B, lq, H, D, generator=g).to(dt).cuda()
    which = torch.randint(0, lk, (B,), generator=g)
    keep = None if mask is None else (torch.arange(lk)[None] == which[:, None]).cuda()
    leaves = [t.requires_grad_(True) for t in (q, k, v, table)]
    out = relative_attention(*leaves, key_mask=keep, q_offset=7)
    dq, dk, dv, dtable = torch.autograd.grad(out, leaves, dout)
    rows = v.detach()[torch.arange(B), :, which].repeat_interleave(H // Hk, 1)[:, None]      # [B, 1, H, D]
    assert torch.equal(out.detach(), rows.expand(-1, lq, -1, -1))
    assert not dq.any() and not dk.any() and not dtable.any(), (dq.abs().max().item(), dk.abs().max().item(), dtable.abs().max().item())
    want = dout.double().sum(1).view(B, Hk, H // Hk, D).sum(2)
    got = dv.double()[torch.arange(B), :, which]
    # P in 16 bits is 1 (f32 carries it 1e-6 off at most); sums of lq H / Hk rows in f32
    assert (got - want).abs().max() <= torch.finfo(dt).eps * want.abs().max() + 2.0 ** -20 * dout.abs().max() * lq


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("L", [40, 300])
def test_the_first_causal_row_passes_no_gradient_through_its_score(L, dtype):
    dt = getattr(torch, dtype)
    g = torch.Generator().manual_seed(L)
    q, k, v = (torch.randn(2, 4, L, 64, generator=g).to(dt).cuda().requires_grad_(True) for _ in range(3))
    table = torch.randn(32, 4, generator=g).cuda()
    out = relative_attention(q, k, v, table, causal=True)
    dq, = torch.autograd.grad(out, q, torch.randn(2, L, 4, 64, generator=g).to(dt).cuda())
    assert not dq[:, :, 0].any() and dq[:, :, 1:].any()
