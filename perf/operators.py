"""Measured cases of the tower operators: attention with a learned relative position bias, the per-head norm of queries and keys with
the position rotation, and the orthogonalised update of an optimizer step.

``run`` computes one pass of a case.  Where ``own`` is false it is the operator's plain form: elementary torch operations in float32
(float64 where 32 bits lose something), rounded once at the end.  Where ``own`` is true it is the call of ``mmlearn_amd`` that a training
or serving program makes.  ``exact`` is the operator's definition in float64, written apart from the plain form.
"""

import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_NS = (3.4445, -4.7750, 2.0315)   # the quintic a X + b (X X^T) X + c (X X^T)^2 X that drives every singular value towards 1


# ---------------------------------------------------------------------------------------------------------------- cases
def _att(name, batch, heads, kv_heads, dim, lq, lk, dtype, train, causal, mask, buckets=32, far=128):
    return {"name": name, "op": "relative_attention", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "lq": lq, "lk": lk,
            "dtype": dtype, "train": train, "causal": causal, "mask": mask, "buckets": buckets, "far": far}


def _qkn(name, batch, length, heads, kv_heads, dim, rot, style, dtype, train, start):
    return {"name": name, "op": "qk_norm_rotary", "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rot": rot, "style": style, "dtype": dtype, "train": train, "start": start}


def _ort(name, count, rows, cols, dtype):
    return {"name": name, "op": "orthogonalize", "count": count, "rows": rows, "cols": cols, "dtype": dtype}


def listed():
    return [
        # one generated token of one sequence against its keys: nothing but latency
        _att("bias decode one", 1, 12, 12, 64, 1, 333, "bf16", False, True, "none"),
        # a serving batch of long sequences of different lengths, one token each, key heads shared by four query heads
        _att("bias decode batch", 32, 32, 8, 128, 1, 8191, "bf16", False, True, "lengths"),
        # captions of a retrieval set through a text tower, inference
        _att("bias captions", 256, 12, 12, 64, 77, 77, "f16", False, False, "lengths"),
        # a text tower trained on documents of ragged length, keep mask of the tokenizer
        _att("bias train documents", 16, 12, 12, 64, 512, 512, "bf16", True, False, "mask"),
        # a causal decoder trained on one long odd length, shared key heads
        _att("bias train long", 2, 16, 4, 128, 4097, 4097, "bf16", True, True, "none"),
        # the queries and keys of one generated token for a small batch
        _qkn("qk token", 8, 1, 12, 12, 64, 64, "half", "bf16", False, 4095),
        # the image tower's tokens, forward and backward
        _qkn("qk train image", 256, 197, 12, 12, 64, 64, "half", "bf16", True, 0),
        # long context with shared key heads, a part of each head rotated, positions far from zero
        _qkn("qk train long", 4, 8192, 32, 8, 128, 64, "interleaved", "bf16", True, 100000),
        # one small matrix of odd size: nothing but latency
        _ort("update small", 1, 201, 65, "f32"),
        # the packed query / key / value weights of a twelve-layer tower
        _ort("update tower", 12, 2304, 768, "f32"),
        # a matrix whose sides fit no tile
        _ort("update odd", 3, 1000, 1777, "bf16"),
        # one large matrix
        _ort("update large", 1, 4096, 4096, "f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("relative_attention", "relative_attention", "qk_norm_rotary", "orthogonalize"))
    if op == "relative_attention":
        kind = rng.choice(("decode", "forward", "train"))
        dim, dtype = rng.choice((64, 128)), rng.choice(("bf16", "f16"))
        kv = rng.choice((1, 2, 4, 8, 12))
        heads = kv * rng.choice((1, 1, 2, 4))
        mask = rng.choice(("none", "lengths", "mask"))
        buckets, far = rng.choice(((32, 128), (32, 128), (64, 256), (16, 40)))
        if kind == "decode":
            lq, lk = rng.choice((1, 1, 1, 4)), _log(rng, 17, 16384)
            batch = min(_log(rng, 1, 64), max(1, 2 ** 27 // (lk * kv * dim)))
            return dict(_att("", batch, heads, kv, dim, lq, lk, dtype, False, True, mask, buckets, far))
        lq = _log(rng, 1, 4096)
        lk = lq if rng.random() < 0.75 else _log(rng, 1, 4096)
        batch = min(_log(rng, 1, 128), max(1, 2 ** 29 // (lq * lk * heads)))
        return dict(_att("", batch, heads, kv, dim, lq, lk, dtype, kind == "train", lq == lk and rng.random() < 0.5, mask, buckets, far))
    if op == "qk_norm_rotary":
        dim = rng.choice((32, 64, 64, 80, 96, 128, 128, 256))
        kv = rng.choice((1, 2, 4, 8, 12))
        heads = kv * rng.choice((1, 1, 2, 4))
        train = rng.random() < 0.6
        length = _log(rng, 1, 8192)
        batch = min(_log(rng, 1, 256), max(1, 2 ** 26 // (length * (heads + kv) * dim)))
        rot = rng.choice((dim, dim, dim // 2, 0))
        return dict(_qkn("", batch, length, heads, kv, dim, rot, rng.choice(("half", "interleaved")), rng.choice(("bf16", "f16", "f32")), train,
                         rng.choice((0, 0, rng.randrange(1, 120000)))))
    rows, cols = _log(rng, 16, 4096), _log(rng, 16, 4096)
    short, wide = min(rows, cols), max(rows, cols)
    count = min(_log(rng, 1, 16), max(1, 2 ** 36 // (short * short * wide)))
    return dict(_ort("", count, rows, cols, rng.choice(("f32", "f32", "bf16", "f16"))))


# ---------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": case}
    if case["op"] == "relative_attention":
        b, h, hk, d, lq, lk = (case[n] for n in ("batch", "heads", "kv_heads", "dim", "lq", "lk"))
        # [B, L, H, D] as a projection leaves them, seen as [B, H, L, D]
        s["q"] = randn(b, lq, h, d).to(dt).transpose(1, 2)
        s["k"] = randn(b, lk, hk, d).to(dt).transpose(1, 2)
        s["v"] = randn(b, lk, hk, d).to(dt).transpose(1, 2)
        s["table"] = randn(case["buckets"], h).to(dt)
        s["mask"] = None
        lengths = torch.randint(max(1, lk // 3), lk + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        if b > 2:
            lengths[b // 2] = 0   # a padded batch ends with samples that hold nothing
        if case["mask"] == "lengths":
            s["mask"] = lengths
        elif case["mask"] == "mask":
            s["mask"] = torch.arange(lk, device="cuda")[None] < lengths[:, None]
        s["offset"] = lk - lq if case["causal"] else 0   # the new tokens are the last ones
        if case["train"]:
            s["dout"] = randn(b, lq, h, d).to(dt)
            for n in ("q", "k", "v", "table"):
                s[n].requires_grad_(True)
    elif case["op"] == "qk_norm_rotary":
        b, l, h, hk, d, rot = (case[n] for n in ("batch", "length", "heads", "kv_heads", "dim", "rot"))
        # the q and k columns of one packed projection
        x = (2.0 * randn(b, l, h + 2 * hk, d)).to(dt)
        s["q"], s["k"] = x[:, :, :h], x[:, :, h:h + hk]
        s["qw"], s["kw"] = ((1.0 + 0.1 * randn(d)).to(dt) for _ in range(2))
        s["positions"] = None
        s["rotary"] = None
        if rot:
            # table of cosines and sines over the positions that a model serves; angles in 64 bits, as far positions need
            last = case["start"] + l
            angle = torch.arange(last, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
                -torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
            s["rotary"] = torch.cat((angle.cos(), angle.sin()), 1).float()
            if case["start"]:
                # each sequence of the batch stands somewhere else
                first = torch.randint(0, case["start"] + 1, (b, 1), generator=g, device="cuda")
                s["positions"] = (first + torch.arange(l, device="cuda")[None]).to(torch.int32)
        if case["train"]:
            s["dq"], s["dk"] = randn(b, l, h, d).to(dt), randn(b, l, hk, d).to(dt)
            s["q"], s["k"] = s["q"].detach().requires_grad_(True), s["k"].detach().requires_grad_(True)
            s["qw"].requires_grad_(True)
            s["kw"].requires_grad_(True)
    else:
        n, r, c = case["count"], case["rows"], case["cols"]
        # a gradient: a few strong directions over noise, small in scale
        rank = max(1, min(r, c) // 32)
        low = randn(n, r, rank) @ randn(n, rank, c) / math.sqrt(rank)
        s["update"] = (1e-3 * (low + 0.5 * randn(n, r, c))).to(dt)
    return s


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _buckets(rel, buckets, far, bidirectional):
    """Bucket of a distance key - query: the nearest distances one by one, farther ones in steps that grow with the logarithm."""
    side = buckets // 2 if bidirectional else buckets
    base = (rel > 0).long() * side if bidirectional else torch.zeros_like(rel)
    dist = rel.abs() if bidirectional else (-rel).clamp(min=0)
    near = side // 2
    steps = torch.log(dist.clamp(min=1).double() / near) / math.log(far / near) * (side - near)
    # 64 bits and a hair of slack: a distance that stands exactly on a border belongs to the bucket that begins there
    log = (near + (steps + 1e-9).floor().long()).clamp(max=side - 1)
    return base + torch.where(dist < near, dist, log)


def _plain_attention(s):
    c = s["case"]
    q, k, v, table = (s[n].detach().float() for n in ("q", "k", "v", "table"))
    dt = s["q"].dtype
    b, h, lq, d = q.shape
    hk, lk = k.shape[1], k.shape[2]
    group = h // hk
    scale = d ** -0.5
    q = q.reshape(b, hk, group, lq, d)
    k, v = k[:, :, None], v[:, :, None]
    rel = torch.arange(lk, device=q.device)[None] - (torch.arange(lq, device=q.device)[:, None] + s["offset"])
    bias = table[_buckets(rel, c["buckets"], c["far"], not c["causal"])]   # [lq, lk, h]
    scores = torch.matmul(q, k.transpose(-1, -2)) * scale + bias.permute(2, 0, 1).reshape(hk, group, lq, lk)
    keep = None
    if s["mask"] is not None:
        m = s["mask"] if s["mask"].dim() == 2 else torch.arange(lk, device=q.device)[None] < s["mask"][:, None]
        keep = m[:, None, None, None]
    if c["causal"]:
        keep = (rel <= 0) if keep is None else keep & (rel <= 0)
    if keep is not None:
        scores = scores.masked_fill(~keep, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)   # a row without a key gives zeros
    out = torch.matmul(p, v).reshape(b, h, lq, d).transpose(1, 2)
    if not c["train"]:
        return {"out": out.to(dt)}
    do = s["dout"].float().transpose(1, 2).reshape(b, hk, group, lq, d)
    dp = torch.matmul(do, v.transpose(-1, -2))
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k).reshape(b, h, lq, d) * scale
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(2) * scale
    # sums over the diagonals of d score: rows of lk + lq read as rows of one more, so that equal distances stand in one column
    w = lk + lq
    skew = torch.nn.functional.pad(ds.sum(0).reshape(h, lq, lk), (0, lq)).reshape(h, lq * w)
    skew = torch.nn.functional.pad(skew, (0, lq)).reshape(h, lq, w + 1).sum(1)
    dist = torch.arange(w + 1, device=q.device)
    dist = torch.where(dist < lk, dist, dist - (w + 1)) - s["offset"]   # the last columns hold the negative distances
    which = _buckets(dist, c["buckets"], c["far"], not c["causal"])
    dtable = torch.matmul((which[None] == torch.arange(c["buckets"], device=q.device)[:, None]).float(), skew.transpose(0, 1))
    return {"out": out.to(dt), "dq": dq.to(dt), "dk": dk.to(dt), "dv": dv.to(dt), "dtable": dtable.to(dt)}


def _turn(x, cos, sin, rot, style, back=False):
    """The rotation of the first ``rot`` columns; ``back``: by the opposite angle."""
    if back:
        sin = -sin
    y = x[..., :rot]
    a, b = (y[..., : rot // 2], y[..., rot // 2:]) if style == "half" else (y[..., 0::2], y[..., 1::2])
    u, w = a * cos - b * sin, b * cos + a * sin
    y = torch.cat((u, w), -1) if style == "half" else torch.stack((u, w), -1).flatten(-2)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_qk(s):
    c = s["case"]
    rot, style, dt = c["rot"], c["style"], s["q"].dtype
    cos = sin = None
    if rot:
        rows = s["rotary"][: c["length"]] if s["positions"] is None else s["rotary"][s["positions"].long()]
        cos, sin = rows[..., None, : rot // 2], rows[..., None, rot // 2:]

    def side(x, w, dy):
        x, w = x.detach().float(), w.detach().float()
        rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        n = x * rstd
        y = n * w
        y = _turn(y, cos, sin, rot, style) if rot else y
        if dy is None:
            return y.to(dt), None, None
        g = dy.float()
        g = _turn(g, cos, sin, rot, style, back=True) if rot else g
        dw = (g * n).double().sum((0, 1, 2))
        gw = g * w
        dx = rstd * (gw - n * (gw * n).mean(-1, keepdim=True))
        return y.to(dt), dx.to(dt), dw.to(dt)

    q, dq, dqw = side(s["q"], s["qw"], s.get("dq"))
    k, dk, dkw = side(s["k"], s["kw"], s.get("dk"))
    return {"q": q, "k": k} if not c["train"] else {"q": q, "k": k, "dq": dq, "dk": dk, "dqw": dqw, "dkw": dkw}


def _plain_orthogonalize(s):
    x = s["update"].float()
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2) if tall else x
    x = x / (x.double().square().sum((1, 2), keepdim=True).sqrt().float() + 1e-7)
    a, b, c = _NS
    for _ in range(5):
        p = torch.matmul(x, x.transpose(1, 2))
        x = a * x + torch.matmul(b * p + c * torch.matmul(p, p), x)
    return (x.transpose(1, 2) if tall else x).to(torch.bfloat16).contiguous()


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    s, c = state, state["case"]
    if not own:
        if c["op"] == "relative_attention":
            return _plain_attention(s)
        return _plain_qk(s) if c["op"] == "qk_norm_rotary" else _plain_orthogonalize(s)
    if c["op"] == "relative_attention":
        from mmlearn_amd.attention import relative_attention

        out = relative_attention(s["q"], s["k"], s["v"], s["table"], max_distance=c["far"], bidirectional=not c["causal"], causal=c["causal"],
                                 key_mask=s["mask"], q_offset=s["offset"])
        if not c["train"]:
            return {"out": out}
        grads = torch.autograd.grad(out, (s["q"], s["k"], s["v"], s["table"]), s["dout"])
        return dict(zip(("out", "dq", "dk", "dv", "dtable"), (out, *grads)))
    if c["op"] == "qk_norm_rotary":
        from mmlearn_amd.attention import qk_norm_rotary

        q, k = qk_norm_rotary(s["q"], s["k"], s["qw"], s["kw"], rotary=s["rotary"], positions=s["positions"],
                              interleaved=c["style"] == "interleaved", eps=1e-6)
        if not c["train"]:
            return {"q": q, "k": k}
        grads = torch.autograd.grad((q, k), (s["q"], s["k"], s["qw"], s["kw"]), (s["dq"], s["dk"]))
        return dict(zip(("q", "k", "dq", "dk", "dqw", "dkw"), (q, k, *grads)))
    from mmlearn_amd.optim import orthogonalize

    return orthogonalize(s["update"], steps=5, coefficients=_NS, eps=1e-7)


# ---------------------------------------------------------------------------------------------------------------- work
def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    if case["op"] == "relative_attention":
        b, h, hk, d, lq, lk = (case[n] for n in ("batch", "heads", "kv_heads", "dim", "lq", "lk"))
        pairs = lq * lk if not case["causal"] else lq * (lk - lq) + lq * (lq + 1) / 2
        if case["mask"] != "none":
            pairs *= 2 / 3   # lengths are spread over the last two thirds
        kv = 2 * b * hk * lk * d * size * (1.0 if case["mask"] == "none" else 2 / 3)
        qo = 2 * b * h * lq * d * size
        if not case["train"]:
            return {"bytes": qo + kv, "flops": 4 * b * h * pairs * d}
        return {"bytes": 2 * (qo + kv), "flops": 14 * b * h * pairs * d}
    if case["op"] == "qk_norm_rotary":
        n = case["batch"] * case["length"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        angles = case["length"] * case["rot"] * 4 * (case["batch"] if case["start"] else 1)
        return {"bytes": n * size * (5 if case["train"] else 2) + angles, "flops": n * (30 if case["train"] else 10)}
    m, n = sorted((case["rows"], case["cols"]))
    # per step: X X^T and its square are symmetric, half of each has to be computed; then the product with X
    return {"bytes": case["count"] * m * n * (size + 2), "flops": 5 * case["count"] * (m * m * n + m ** 3 + 2 * m * m * n)}


# ---------------------------------------------------------------------------------------------------------------- definition in 64 bits
def _border_table(case):
    """The bucket of every distance 0 .. far by integer arithmetic: a step is reached when (dist / near)^(side - near) >= (far / near)^t."""
    side = case["buckets"] if case["causal"] else case["buckets"] // 2
    near, far = side // 2, case["far"]
    got = []
    for dist in range(far + 1):
        t = 0
        while dist >= near and t < side - near - 1 and dist ** (side - near) * near ** (t + 1) >= far ** (t + 1) * near ** (side - near):
            t += 1
        got.append(dist if dist < near else near + t)
    return torch.tensor(got, device="cuda"), side


def _exact_attention(s, case):
    b, h, hk, d, lq, lk = (case[n] for n in ("batch", "heads", "kv_heads", "dim", "lq", "lk"))
    if 16 * b * h * lq * lk * d > 3e13:
        return None
    q, k, v, table = (s[n].detach().double() for n in ("q", "k", "v", "table"))
    steps, side = _border_table(case)
    i = torch.arange(lq, device="cuda") + s["offset"]
    j = torch.arange(lk, device="cuda")
    back = i[:, None] - j[None]
    bucket = steps[back.abs().clamp(max=case["far"])]
    if case["causal"]:
        bucket = torch.where(back < 0, 0, bucket)
    else:
        bucket = torch.where(back < 0, bucket + side, bucket)
    out = torch.zeros(b, lq, h, d, dtype=torch.float64, device="cuda")
    grads = {"dq": torch.zeros(b, h, lq, d, dtype=torch.float64, device="cuda"), "dk": torch.zeros(b, hk, lk, d, dtype=torch.float64, device="cuda"),
             "dv": torch.zeros(b, hk, lk, d, dtype=torch.float64, device="cuda"), "dtable": torch.zeros(case["buckets"], h, dtype=torch.float64, device="cuda")}
    lengths = s["mask"]
    for head in range(h):
        kh = head // (h // hk)
        bias = table[:, head][bucket]
        total = torch.zeros(lq, lk, dtype=torch.float64, device="cuda") if case["train"] else None
        for n in range(0, b, max(1, 2 ** 26 // (lq * lk))):
            e = min(b, n + max(1, 2 ** 26 // (lq * lk)))
            valid = torch.ones(e - n, lq, lk, dtype=torch.bool, device="cuda")
            if lengths is not None:
                valid &= (lengths[n:e] if lengths.dim() == 2 else j[None] < lengths[n:e, None])[:, None]
            if case["causal"]:
                valid &= (back >= 0)[None]
            z = torch.einsum("bid,bjd->bij", q[n:e, head], k[n:e, kh]) / math.sqrt(d) + bias
            z = torch.where(valid, z, torch.full_like(z, -1e300))
            p = torch.where(valid, torch.exp(z - z.max(-1, keepdim=True).values), torch.zeros_like(z))
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            out[n:e, :, head] = torch.einsum("bij,bjd->bid", p, v[n:e, kh])
            if case["train"]:
                g = s["dout"][n:e, :, head].double()
                t = torch.einsum("bid,bjd->bij", g, v[n:e, kh])
                t = p * (t - (t * p).sum(-1, keepdim=True))
                grads["dq"][n:e, head] = torch.einsum("bij,bjd->bid", t, k[n:e, kh]) / math.sqrt(d)
                grads["dk"][n:e, kh] += torch.einsum("bij,bid->bjd", t, q[n:e, head]) / math.sqrt(d)
                grads["dv"][n:e, kh] += torch.einsum("bij,bid->bjd", p, g)
                total += t.sum(0)
        if case["train"]:
            for w in range(case["buckets"]):
                grads["dtable"][w, head] = total[bucket == w].sum()
    return {"out": out, **grads} if case["train"] else {"out": out}


def _exact_qk(s, case):
    rot = case["rot"]
    place = torch.arange(case["length"], device="cuda")[None] if s["positions"] is None else s["positions"].long()
    got = {}
    for n in ("q", "k"):
        x, w = s[n].detach().double().requires_grad_(True), s[n + "w"].detach().double().requires_grad_(True)
        y = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case["dim"] + 1e-6) * w
        if rot:
            angles = s["rotary"].double()[place]
            z = torch.complex(angles[..., : rot // 2], angles[..., rot // 2:])[:, :, None]
            y0 = y[..., :rot]
            y0 = y0.unflatten(-1, (2, rot // 2)).transpose(-1, -2) if case["style"] == "half" else y0.unflatten(-1, (rot // 2, 2))
            t = torch.view_as_real(torch.view_as_complex(y0.contiguous()) * z)
            t = t.transpose(-1, -2) if case["style"] == "half" else t
            y = torch.cat((t.flatten(-2), y[..., rot:]), -1)
        got[n] = y.detach()
        if case["train"]:
            got["d" + n], got["d" + n + "w"] = torch.autograd.grad(y, (x, w), s["d" + n].double())
    return got


def _exact_orthogonalize(s, case):
    m, n = sorted((case["rows"], case["cols"]))
    got = []
    for g in s["update"].double():
        x = g.T if case["rows"] > case["cols"] else g
        x = x / (torch.linalg.norm(x) + 1e-7)
        for _ in range(5):
            p = x @ x.T
            x = _NS[0] * x + _NS[1] * (p @ x) + _NS[2] * (p @ (p @ x))
        got.append(x.T if case["rows"] > case["cols"] else x)
    return torch.stack(got)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "relative_attention":
        return _exact_attention(s, case)
    return _exact_qk(s, case) if case["op"] == "qk_norm_rotary" else _exact_orthogonalize(s, case)
