"""Short-sequence self-attention on MI355X (second step).

``attention(q, k, v, scale, dropout_p)`` = ``dropout(softmax(scale * q k^T + mask)) v`` for ``[B, H, L, 64]`` bf16 operands with
``L <= 256`` -- the shape of every attention call in the encoders of the headline workload (ViT-B/16 L = 197, mmlearn's own ViT
L = 196 / 169, BERT L = 77 with attention dropout 0.1 and the tokenizer's key-padding mask).  One workgroup keeps a whole
(batch, head) problem on chip (``csrc/attention.hip``); the dropout mask is a counter-based function of a per-call seed
drawn from torch's CPU generator (so ``torch.manual_seed`` reproduces it), regenerated in the backward.  The mask is a per-sample
KEY mask (``key_bias``: the records of :func:`key_bias_of`, one per batch, shared by all layers) and / or the causal triangle.
Registered with HF transformers' ``AttentionInterface`` as ``"mmlearn_hip"`` so that ``CLIPVisionModel`` / ``BertModel`` & co. can
select it per config; calls it cannot serve (a mask that is not provably a key-padding mask, other head dims or dtypes) are
forwarded to SDPA unchanged.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad

from . import kernels as K


def supported(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, attention_mask=None, dropout: float = 0.0, is_causal=False) -> bool:
    """Operand test of the kernels.  ``attention_mask``: None, or a mask :func:`key_mask_view` proves to be a key-padding mask."""
    return (q.is_cuda and q.dtype == torch.bfloat16 and k.dtype == torch.bfloat16 and v.dtype == torch.bfloat16 and q.dim() == 4
            and q.shape == k.shape == v.shape and q.shape[-1] == 64 and q.shape[-2] <= 256
            and (attention_mask is None or key_mask_view(attention_mask, q.shape[0], q.shape[2]) is not None)
            and 0.0 <= float(dropout) < 1.0 and q.stride(-1) == 1 and k.stride(-1) == 1 and v.stride(-1) == 1
            and all(s % 8 == 0 for t in (q, k, v) for s in t.stride()[:3]))


def key_mask_view(mask: torch.Tensor, B: int, L: int):
    """``(view [B, L], additive)`` when the SHAPE AND STRIDES of ``mask`` prove it masks keys only -- the same row for every head and
    every query: ``[B, L]``, ``[B, 1, 1, L]``, or ``[B, 1, Lq, L]`` / ``[B, H, Lq, L]`` expanded along the broadcast dims (stride 0).  A
    materialised ``[B, 1, L, L]`` tensor (what HF's mask helpers hand to the attention modules) could hold anything and is refused
    (None): ``fused.py`` knows where such a tensor came from and keeps the 2-D mask instead.  ``additive``: a floating mask in logit
    units (0 / ``finfo.min``) as opposed to a boolean / integer keep-mask."""
    if not isinstance(mask, torch.Tensor) or not mask.is_cuda or mask.shape[0] != B or mask.shape[-1] != L or mask.stride(-1) != 1 and L > 1:
        return None
    if mask.dim() == 4:
        if not all(mask.shape[d] == 1 or mask.stride(d) == 0 for d in (1, 2)):
            return None
        mask = mask[:, 0, 0]
    elif mask.dim() != 2:
        return None
    if mask.dtype in (torch.bool, torch.uint8, torch.int32, torch.int64):
        return mask, False
    if mask.dtype in (torch.float32, torch.bfloat16):
        return mask, True
    return None


def key_bias_of(mask, B: int, L: int, additive: Optional[bool] = None):
    """Key bias records (``kernels.attn_key_bias``) of a mask :func:`key_mask_view` accepts; None otherwise.  A 2-D floating mask is a
    KEEP mask (HF's ``attention_mask`` of ones and zeros) unless ``additive`` says otherwise; a 4-D floating mask is additive."""
    dim = mask.dim() if isinstance(mask, torch.Tensor) else 0
    kv = key_mask_view(mask, B, L)
    if kv is None:
        return None
    view, add = kv
    if additive is None:
        additive = add and dim == 4
    if view.stride(0) < L:   # expanded over the batch as well
        view = view.contiguous()
    if view.dtype == torch.bfloat16 and not additive:
        view = view.float()
    return K.attn_key_bias(view, additive=bool(additive and view.is_floating_point()))


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, dropout_p, seed, key_bias=None, causal=False):
        out, lse = K.attn_fwd(q, k, v, scale, dropout_p, seed, key_bias, causal)   # out: [B, L, H, 64] contiguous
        ctx.save_for_backward(q, k, v, out, lse, key_bias)
        ctx.scale, ctx.dropout_p, ctx.seed, ctx.causal = scale, dropout_p, seed, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse, key_bias = ctx.saved_tensors
        dq, dk, dv = K.attn_bwd(q, k, v, out, lse, dout.contiguous(), ctx.scale, ctx.dropout_p, ctx.seed, key_bias=key_bias, causal=ctx.causal)
        return dq, dk, dv, None, None, None, None, None


class _AttentionPacked(torch.autograd.Function):
    """Same kernels on a packed ``[B, L, 3, H, 64]`` QKV tensor (the output of ONE fused projection); the backward writes
    dq / dk / dv straight into one packed gradient, so autograd sees a single tensor in and out."""

    @staticmethod
    def forward(ctx, qkv, scale, dropout_p, seed, key_bias=None, causal=False):
        q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))   # [B, H, L, 64] views, row stride 3*H*64
        out, lse = K.attn_fwd(q, k, v, scale, dropout_p, seed, key_bias, causal)
        ctx.save_for_backward(qkv, out, lse, key_bias)
        ctx.scale, ctx.dropout_p, ctx.seed, ctx.causal = scale, dropout_p, seed, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        qkv, out, lse, key_bias = ctx.saved_tensors
        q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
        return (K.attn_bwd(q, k, v, out, lse, dout.contiguous(), ctx.scale, ctx.dropout_p, ctx.seed, packed=True, key_bias=key_bias,
                           causal=ctx.causal), None, None, None, None, None)


def _causal_bias(key_bias, causal: bool, like: torch.Tensor, B: int, L: int):
    """The kernels take the causal triangle only together with a key bias record: an all-attended one when there is no padding."""
    if causal and key_bias is None:
        key_bias = K.attn_key_bias(torch.full((B,), L, dtype=torch.int32, device=like.device), L=L)
    return key_bias


def attention_qkvpacked(qkv: torch.Tensor, scale: Optional[float] = None, dropout_p: float = 0.0, seed: Optional[int] = None,
                        key_bias: Optional[torch.Tensor] = None, causal: bool = False) -> torch.Tensor:
    """``qkv``: ``[B, L, 3, H, 64]`` bf16 contiguous (``Linear(E, 3E)(x).view(B, L, 3, H, 64)``) -> ``[B, L, H, 64]``.
    ``key_bias``: :func:`key_bias_of` records of a key-padding mask; ``causal``: also mask key j > query i."""
    K.require_gpu(qkv)
    if not (qkv.dim() == 5 and qkv.shape[2] == 3 and qkv.shape[-1] == 64 and qkv.shape[1] <= 256 and qkv.dtype == torch.bfloat16
            and qkv.is_contiguous() and 0.0 <= dropout_p < 1.0):
        raise ValueError("mmlearn_amd.attention_qkvpacked: need a contiguous bf16 [B, L<=256, 3, H, 64] tensor")
    if dropout_p > 0.0 and seed is None:
        seed = draw_seed()
    key_bias = _causal_bias(key_bias, causal, qkv, qkv.shape[0], qkv.shape[1])
    return _AttentionPacked.apply(qkv, float(scale if scale is not None else 0.125), float(dropout_p), int(seed or 0), key_bias, bool(causal))


def draw_seed() -> int:
    """A 63-bit seed from torch's default CPU generator (no device sync; reproducible under ``torch.manual_seed``)."""
    return int(torch.empty((), dtype=torch.int64).random_().item())


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None, dropout_p: float = 0.0,
              seed: Optional[int] = None, key_bias: Optional[torch.Tensor] = None, causal: bool = False) -> torch.Tensor:
    """q, k, v: ``[B, H, L, 64]`` bf16 (any strides with a contiguous last dim).  Returns ``[B, L, H, 64]`` contiguous,
    i.e. already in the layout the output projection wants (``.reshape(B, L, H*64)`` is free).  ``dropout_p`` drops
    attention probabilities (training-time semantics of ``F.scaled_dot_product_attention(dropout_p=...)``).  ``key_bias``: the
    records of :func:`key_bias_of` for a key-padding mask (``attn_mask=[B, 1, 1, L]`` of SDPA); ``causal`` = ``is_causal``."""
    K.require_gpu(q)
    if not supported(q, k, v, dropout=dropout_p):
        raise ValueError("mmlearn_amd.attention: need bf16 [B, H, L<=256, 64] operands with contiguous last dim")
    if dropout_p > 0.0 and seed is None:
        seed = draw_seed()
    key_bias = _causal_bias(key_bias, causal, q, q.shape[0], q.shape[2])
    return _Attention.apply(q, k, v, float(scale if scale is not None else q.shape[-1] ** -0.5), float(dropout_p), int(seed or 0), key_bias,
                            bool(causal))


def hf_attention_forward(module, query, key, value, attention_mask, dropout: float = 0.0, scaling: Optional[float] = None,
                         is_causal: Optional[bool] = None, **kwargs):
    """transformers ``AttentionInterface`` entry: same contract as ``sdpa_attention_forward`` (returns
    ``(attn_output [B, L, H, dh], None)``).  Unsupported calls fall through to SDPA."""
    if supported(query, key, value, attention_mask, dropout, bool(is_causal)):
        kb = None if attention_mask is None else key_bias_of(attention_mask, query.shape[0], query.shape[2])
        return attention(query, key, value, scaling, float(dropout), key_bias=kb, causal=bool(is_causal)), None
    from transformers.integrations.sdpa_attention import sdpa_attention_forward

    return sdpa_attention_forward(module, query, key, value, attention_mask, dropout=dropout, scaling=scaling, is_causal=is_causal, **kwargs)


def register_hf_attention(name: str = "mmlearn_hip") -> str:
    """Make ``config._attn_implementation = "mmlearn_hip"`` available to HF models."""
    from transformers import AttentionInterface

    AttentionInterface.register(name, hf_attention_forward)
    return name


# ------------------------------------------------------------------ per-head norm of queries and keys with the position rotation
def rotary_table(positions: int, dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """f32 ``[positions, dim]`` table for :func:`qk_norm_rotary`: ``dim / 2`` cosines, then ``dim / 2`` sines, of the angles
    ``position * base ** (-2 i / dim)``, formed in float64 (in float32 the angle of position 100,000 is off by thousandths of a turn)."""
    if positions < 0 or dim < 0 or dim % 2 or not base > 0:
        raise ValueError("mmlearn_amd.rotary_table: need positions >= 0, an even dim >= 0 and base > 0")
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64) / max(dim, 1))
    return torch.cat((angle.cos(), angle.sin()), 1).float().to(device)


def _records(*operands: Optional[torch.Tensor]) -> bool:
    """Whether autograd has to see the call (an autograd function costs a single token more than its kernel): to record it, or, within a
    level of forward-mode differentiation, to refuse operands with a tangent, which do not require grad (past the function their
    derivative would vanish without a word)."""
    return forward_ad._current_level >= 0 or (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in operands))


class _QKNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, table, positions, interleaved, eps):
        ctx.save_for_backward(q, k, qw, kw, table, positions)
        ctx.interleaved, ctx.eps = interleaved, eps
        return K.qk_norm_rotary_fwd(q, k, qw, kw, table, positions, interleaved, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dqo, dko):
        q, k, qw, kw, table, positions = ctx.saved_tensors
        dqo, dko = (g if g.stride(-1) == 1 or g.shape[-1] == 1 else g.contiguous() for g in (dqo.to(q.dtype), dko.to(k.dtype)))
        grads = K.qk_norm_rotary_bwd(q, k, qw, kw, table, positions, dqo, dko, ctx.interleaved, ctx.eps, ctx.needs_input_grad[2],
                                     ctx.needs_input_grad[3])
        return (*grads, None, None, None, None)


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                   rotary: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, interleaved: bool = False,
                   eps: float = 1e-6):
    """Per-head RMS norm of queries and keys and the rotation by their positions, one launch forward and one (plus the sum of the weights'
    gradients) backward.  ``q`` ``[B, L, H, D]`` and ``k`` ``[B, L, Hk, D]`` (f32 / bf16 / f16, any strides with a contiguous last dim --
    slices of a packed projection --, ``D`` even, at most 256) -> contiguous ``(q', k')`` of the same shapes, with
    ``q' = R(position) (q_weight * q / sqrt(mean(q ** 2) + eps))``.  Weights: ``[D]``, f32 or of the operands' type, None = ones.
    ``rotary``: a :func:`rotary_table` of even width ``<= D``; of a head's first ``rotary.shape[1]`` values the pairs ``(i, i + width / 2)``
    turn (``interleaved``: ``(2 i, 2 i + 1)``), the others pass.  None: no rotation.  ``positions``: int32 / int64 ``[L]`` or ``[B, L]``, rows of
    the table; None: ``0 .. L - 1``.  They are read on the device: a position outside the table makes its rows NaN.
    Forward-mode derivatives are refused.  Both passes may be captured into a HIP graph.  As with every autograd function, no output of an
    eager pass over the same leaves may be alive then: it would keep the leaves' gradient nodes on that pass's stream.
    ``torch.compile`` does not trace the call: the graph breaks around it."""
    if torch.compiler.is_dynamo_compiling():
        return _qk_norm_rotary_untraced(q, k, q_weight, k_weight, rotary, positions, interleaved, eps)
    K.require_gpu(q, "query")
    name = "mmlearn_amd.qk_norm_rotary"
    if not (q.dim() == k.dim() == 4 and q.shape[:2] == k.shape[:2] and q.shape[3] == k.shape[3] and q.dtype == k.dtype
            and q.dtype in (torch.float32, torch.bfloat16, torch.float16)):
        raise ValueError(f"{name}: need q [B, L, H, D] and k [B, L, Hk, D] of one type (float32, bfloat16 or float16)")
    B, L, _, D = q.shape
    if D % 2 or not 2 <= D <= 256 or any(t.stride(3) != 1 for t in (q, k)):
        raise ValueError(f"{name}: the head dim must be even, at most 256, and contiguous")
    for w in (q_weight, k_weight):
        if w is not None and not (w.shape == (D,) and w.is_contiguous() and w.dtype in (torch.float32, q.dtype)):
            raise ValueError(f"{name}: weights are contiguous [D] tensors, float32 or of the operands' type")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError(f"{name}: both weights must have one type")
    if rotary is not None:
        if not (rotary.dim() == 2 and rotary.dtype == torch.float32 and rotary.is_contiguous() and rotary.shape[1] % 2 == 0
                and rotary.shape[1] <= D and not rotary.requires_grad):
            raise ValueError(f"{name}: rotary is a contiguous float32 [positions, width] table without gradient, its width even and at most the head dim")
        if positions is None and rotary.shape[0] < L:
            raise ValueError(f"{name}: the rotary table holds {rotary.shape[0]} positions, the sequence has {L}")
        if rotary.shape[1] == 0:
            rotary = None
    elif positions is not None:
        raise ValueError(f"{name}: positions are rows of a rotary table, and there is none")
    if rotary is None:
        positions = None
    if positions is not None and not (positions.dtype in (torch.int32, torch.int64) and tuple(positions.shape) in ((L,), (B, L))
                                      and (L <= 1 or positions.stride(-1) == 1)):
        raise ValueError(f"{name}: positions are int32 or int64 [L] or [B, L] with a contiguous last dim")
    if any(t is not None and t.device != q.device for t in (k, q_weight, k_weight, rotary, positions)):
        raise ValueError(f"{name}: all operands must be on one device")
    if not _records(q, k, q_weight, k_weight):
        return K.qk_norm_rotary_fwd(q, k, q_weight, k_weight, rotary, positions, interleaved, eps)
    return _QKNormRotary.apply(q, k, q_weight, k_weight, rotary, positions, bool(interleaved), float(eps))


_qk_norm_rotary_untraced = torch.compiler.disable(qk_norm_rotary)


# ------------------------------------------------------------------ attention with a learned relative position bias
def _places(*operands: Optional[torch.Tensor]):
    return [t if t is None else (t.data_ptr(), t.stride()) for t in operands]


class _RelativeAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, key_mask, offsets, how):
        p = K.rel_attn_operands(q, k, v, table, *how[:4], key_mask, how[4] if offsets is None else offsets)
        out, out_lo, lse = K.rel_attn_fwd(p, q, True)
        ctx.save_for_backward(q, k, v, table, key_mask, offsets, out, out_lo, lse)
        ctx.how, ctx.operands, ctx.places = how, p, _places(q, k, v, table, key_mask, offsets)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, table, key_mask, offsets, out, out_lo, lse = ctx.saved_tensors
        p, how = ctx.operands, ctx.how
        if ctx.places != _places(q, k, v, table, key_mask, offsets):   # (hooks on saved tensors brought them back elsewhere)
            p = K.rel_attn_operands(q, k, v, table, *how[:4], key_mask, how[4] if offsets is None else offsets)
        dout = dout.to(q.dtype).contiguous()
        if dout.data_ptr() % 16:
            dout = dout.clone()
        grads = K.rel_attn_bwd(p, q, k, table, out, out_lo, lse, dout, ctx.needs_input_grad[3])
        return (*grads, None, None, None)


def relative_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, max_distance: int = 128, bidirectional: bool = True,
                       scale: Optional[float] = None, causal: bool = False, key_mask: Optional[torch.Tensor] = None, q_offset=0):
    """``softmax(scale * q k^T + table[bucket(j - i)]) v`` with a learned bias per head for each bucket of distances (key minus query), and
    its gradients, the table's included.  ``q`` ``[B, H, Lq, D]``, ``k`` / ``v`` ``[B, Hk, Lk, D]``: bf16 or f16, ``D`` 64 or 128, ``H`` a multiple
    of ``Hk`` (key heads shared by neighbouring query heads), any lengths, any strides that are multiples of 8 with a contiguous last dim.
    Returns ``[B, Lq, H, D]`` contiguous.

    ``table`` ``[buckets, H]``, f32 or of the operands' type (HF's ``relative_attention_bias.weight``).  With ``bidirectional`` the first half of
    the buckets serves keys at or before the query, the second half keys behind it; otherwise keys behind it count as distance 0.  Of a
    side's buckets (at least 2, at most 128) the first half holds one distance each, the others widen with the logarithm up to
    ``max_distance`` (above the number of single distances where there are more than two, at most 512), beyond which all distances share the last one.

    ``key_mask``: ``[B, Lk]`` bool / uint8 / int32 / int64 with nonzero = attended, or int32 / int64 ``[B]`` numbers of leading keys.  What masked
    keys and values hold does not matter.  ``causal``: only keys ``j <= i + q_offset``; what stands behind the last query (the free places of a
    cache) does not matter either, but a NaN or an infinity in a key or value of the queries' own stretch may reach earlier rows near it.
    ``q_offset``: position of query 0 among the keys, an int or an int32 tensor ``[B]`` (one token against a cache: the number of keys before
    it).  A row that nothing is left for gives zeros and passes no gradient.

    A call that autograd records sums its result from weights in two 16-bit parts, one that it does not from weights rounded once (with few rows a
    key head both do the former): the same value within the type's rounding, not bit for bit.
    The table's gradient is exact to about 1e-5 of its size before it is rounded to the table's type; forward-mode derivatives are
    refused.  A HIP graph may hold both passes if no output of an eager pass over the same leaves is alive.  ``torch.compile`` does not trace the
    call: the graph breaks around it."""
    if torch.compiler.is_dynamo_compiling():   # (the kernels' descriptions are ctypes structures, which a resumed trace takes for their classes)
        return _relative_attention_untraced(q, k, v, table, max_distance, bidirectional, scale, causal, key_mask, q_offset)
    K.require_gpu(q, "query")
    name = "mmlearn_amd.relative_attention"
    if not (q.dim() == k.dim() == v.dim() == 4 and q.dtype in (torch.bfloat16, torch.float16) and q.dtype == k.dtype == v.dtype):
        raise ValueError(f"{name}: need 4-dimensional q, k, v of one type, bfloat16 or float16")
    B, H, _, D = q.shape
    if not (k.shape == v.shape and k.shape[0] == B and k.shape[3] == D and D in (64, 128) and k.shape[1] >= 1 and H >= 1 and H % k.shape[1] == 0):
        raise ValueError(f"{name}: need q [B, H, Lq, D], k and v [B, Hk, Lk, D], D 64 or 128, H a multiple of Hk")
    for t in (q, k, v):
        b, h, row = K._strides_bhl(t)
        if t.stride(3) != 1 or (b | h | row) % 8 or t.data_ptr() % 16 or row > 1 << 23:
            raise ValueError(f"{name}: operands need a contiguous last dim, strides that are multiples of 8 (rows: at most 2^23) and 16-byte alignment")
    if max(q.shape[2], k.shape[2]) > 1 << 28:
        raise ValueError(f"{name}: at most 2^28 rows")
    buckets = table.shape[0] if table.dim() == 2 else 0
    if not (table.dim() == 2 and table.shape[1] == H and table.is_contiguous() and table.dtype in (torch.float32, q.dtype)):
        raise ValueError(f"{name}: table is a contiguous [buckets, H] tensor, float32 or of the operands' type")
    side = buckets // 2 if bidirectional else buckets
    if not 2 <= side <= 128 or (bidirectional and buckets % 2):
        raise ValueError(f"{name}: need 2 to 128 buckets a side, an even number of them if bidirectional; got {buckets}")
    least = side // 2 + (side > 2)   # (two buckets a side: distance 0 and the rest, no logarithm)
    if not (isinstance(max_distance, int) and least <= max_distance <= 512):
        raise ValueError(f"{name}: max_distance must be an int of at least {least} and at most 512")
    if key_mask is not None:
        if (key_mask.dim(), key_mask.dtype) not in K._REL_MASKS or tuple(key_mask.shape) != ((B,) if key_mask.dim() == 1 else (B, k.shape[2])):
            raise ValueError(f"{name}: key_mask is [B, Lk] bool / uint8 / int32 / int64, or int32 / int64 [B] lengths")
        if key_mask.shape[-1] > 1 and key_mask.stride(-1) != 1:
            raise ValueError(f"{name}: key_mask needs a contiguous last dim")
    offsets = q_offset if isinstance(q_offset, torch.Tensor) else None
    if offsets is not None and not (offsets.dtype == torch.int32 and offsets.shape == (B,) and offsets.is_contiguous()):
        raise ValueError(f"{name}: q_offset is an int or a contiguous int32 [B] tensor")
    if offsets is None and not (isinstance(q_offset, int) and abs(q_offset) < 1 << 29):
        raise ValueError(f"{name}: q_offset is an int below 2^29 in size, or an int32 [B] tensor")
    if any(t is not None and t.device != q.device for t in (k, v, table, key_mask, offsets)):
        raise ValueError(f"{name}: all operands must be on one device")
    scale = D ** -0.5 if scale is None else float(scale)
    how = max_distance, bool(bidirectional), scale, bool(causal), 0 if offsets is not None else q_offset
    if not _records(q, k, v, table):
        return K.rel_attn_fwd(K.rel_attn_operands(q, k, v, table, *how[:4], key_mask, q_offset), q, False)[0]
    return _RelativeAttention.apply(q, k, v, table, key_mask, offsets, how)


_relative_attention_untraced = torch.compiler.disable(relative_attention)
