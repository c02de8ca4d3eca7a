"""Attention mechanisms.

Capability parity with /root/reference/npf/architectures/attention.py
(factory :16-86; BaseAttender :89-169; DotAttender :172-220; Multiplicative
:223-258; Additive :261-302; Cosine :305-322; Distance :325-372; Multihead
:375-527; Transformer :530-588).

MI355X-first: the hot scaled-dot path (softmax over keys + value reduction)
dispatches to the fused CDNA4 HIP kernel via `npf.ops.attention_qkv`; the
surrounding projections stay hipBLASLt GEMMs.  Head split/merge is a pure
layout choice and is kept identical to the reference so checkpoints and
numerics match.
"""

import abc
import math

import torch
import torch.nn as nn
from torch.nn.modules.distance import CosineSimilarity

from npf.ops import functional as ops
from npf.utils.initialization import weights_init

from .mlp import MLP

__all__ = ["get_attender"]

_STR_ATTENDERS = {}


def get_attender(attention, kq_size, value_size, out_size, **kwargs):
    """Build an attender by name or callable (reference attention.py:16-86).

    Supported names: multiplicative, additive, scaledot, cosine, manhattan,
    euclidean, weighted_dist, multihead, transformer, differential,
    differential_transformer.
    """
    if not isinstance(attention, str):
        return attention(kq_size, value_size, out_size, **kwargs)

    attention = attention.lower()
    try:
        factory = _STR_ATTENDERS[attention]
    except KeyError:
        raise ValueError(f"Unknown attention method {attention}")
    return factory(kq_size, value_size, out_size, **kwargs)


def _register(name, **preset):
    def deco(cls):
        _STR_ATTENDERS[name] = lambda *a, **kw: cls(*a, **preset, **kw)
        return cls

    return deco


class BaseAttender(abc.ABC, nn.Module):
    """Shared attender skeleton: score -> (softmax) -> value sum -> resize.

    Reference: attention.py:89-169.
    """

    def __init__(self, kq_size, value_size, out_size, is_normalize=True, dropout=0):
        super().__init__()
        self.kq_size = kq_size
        self.value_size = value_size
        self.out_size = out_size
        self.is_normalize = is_normalize
        self.dropout = nn.Dropout(p=dropout) if dropout > 0 else nn.Identity()
        self.is_resize = self.value_size != self.out_size
        if self.is_resize:
            self.resizer = nn.Linear(self.value_size, self.out_size)
        self.reset_parameters()

    def reset_parameters(self):
        weights_init(self)

    def _fusable(self, keys, queries):
        """Whether the fused softmax+bmm HIP path applies."""
        return (
            self.is_normalize
            and isinstance(self.dropout, nn.Identity)
            and keys.dim() == 3
            and queries.dim() == 3
        )

    def forward(self, keys, queries, values, **kwargs):
        """keys [B,K,kq], queries [B,Q,kq], values [B,K,v] -> [B,Q,out]."""
        context = self._attend(keys, queries, values, **kwargs)
        if self.is_resize:
            context = self.resizer(context)
        return context

    def _attend(self, keys, queries, values, **kwargs):
        logits = self.score(keys, queries, **kwargs)
        attn = logits.softmax(dim=-1) if self.is_normalize else logits
        attn = self.dropout(attn)
        return torch.bmm(attn, values)

    @abc.abstractmethod
    def score(self, keys, queries, **kwargs):
        """Return logits [B, Q, K]."""


@_register("scaledot", is_scale=True)
class DotAttender(BaseAttender):
    """(Scaled) dot-product attention (reference attention.py:172-220)."""

    def __init__(self, *args, is_scale=True, **kwargs):
        super().__init__(*args, **kwargs)
        self.is_scale = is_scale

    def score(self, keys, queries):
        # 4-D keys arise on the relative-position path (one key set per query)
        keys_shape = "bqkd" if keys.dim() == 4 else "bkd"
        queries_shape = "bqkd" if queries.dim() == 4 else "bqd"
        logits = torch.einsum(f"{keys_shape},{queries_shape}->bqk", keys, queries)
        if self.is_scale:
            logits = logits / math.sqrt(queries.size(-1))
        return logits

    def _attend(self, keys, queries, values, **kwargs):
        if self._fusable(keys, queries) and not kwargs:
            scale = 1.0 / math.sqrt(queries.size(-1)) if self.is_scale else 1.0
            return ops.attention_qkv(keys, queries, values, scale)
        return super()._attend(keys, queries, values, **kwargs)


@_register("multiplicative")
class MultiplicativeAttender(BaseAttender):
    """Multiplicative (Luong) attention (reference attention.py:223-258)."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        self.linear = nn.Linear(self.kq_size, self.kq_size, bias=False)
        self.dot = DotAttender(*args, is_scale=False)
        self.reset_parameters()

    def score(self, keys, queries):
        return self.dot.score(keys, self.linear(queries))


@_register("additive")
class AdditiveAttender(BaseAttender):
    """Additive (Bahdanau) attention (reference attention.py:261-302)."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        self.mlp = MLP(self.kq_size * 2, 1, hidden_size=self.kq_size, activation=nn.Tanh())
        self.reset_parameters()

    def score(self, keys, queries):
        batch_size, n_queries, kq_size = queries.shape
        n_keys = keys.size(1)
        keys = keys.unsqueeze(1).expand(batch_size, n_queries, n_keys, kq_size)
        queries = queries.unsqueeze(2).expand(batch_size, n_queries, n_keys, kq_size)
        return self.mlp(torch.cat((keys, queries), dim=-1)).squeeze(-1)


@_register("cosine")
class CosineAttender(BaseAttender):
    """Cosine-similarity attention (reference attention.py:305-322)."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        self.similarity = CosineSimilarity(dim=1)

    def score(self, keys, queries):
        batch_size, n_queries, kq_size = queries.shape
        n_keys = keys.size(1)
        keys = keys.view(batch_size, kq_size, 1, n_keys)
        queries = queries.view(batch_size, kq_size, n_queries, 1)
        return self.similarity(keys, queries)


@_register("manhattan", p=1)
@_register("euclidean", p=2)
@_register("weighted_dist", p=1, is_weight=True)
class DistanceAttender(BaseAttender):
    """Negative (weighted) distance attention (reference attention.py:325-372)."""

    def __init__(self, *args, p=1, is_weight=False, **kwargs):
        super().__init__(*args, **kwargs)
        self.p = p
        self.is_weight = is_weight
        if self.is_weight:
            self.weighter = nn.Linear(self.kq_size, self.kq_size)
        self.reset_parameters()

    def score(self, keys, queries):
        diff = keys.unsqueeze(1) - queries.unsqueeze(2)
        if self.is_weight:
            diff = self.weighter(diff)
        return -torch.norm(diff, p=self.p, dim=-1) ** 2


@_register("multihead")
class MultiheadAttender(nn.Module):
    """Multi-head scaled-dot attention (reference attention.py:375-527).

    The k/q/v projections are single [kq, kq] linears (head split afterwards),
    head stacking is head-major ([h*B + b]), and `value_head_size` follows the
    reference's `kq_size // n_heads` definition (attention.py:432).  All of
    this is checkpoint-format-relevant.  The inner softmax(QK^T/sqrt(d))V runs
    on the fused HIP kernel through `DotAttender._attend`.
    """

    def __init__(
        self,
        kq_size,
        value_size,
        out_size,
        n_heads=8,
        is_post_process=True,
        dropout=0,
        is_relative_pos=False,
    ):
        super().__init__()
        self.is_relative_pos = is_relative_pos
        self.key_transform = nn.Linear(kq_size, kq_size, bias=False)
        self.query_transform = nn.Linear(kq_size, kq_size, bias=not is_relative_pos)
        self.value_transform = nn.Linear(value_size, value_size, bias=False)
        self.dot = DotAttender(kq_size, value_size, out_size, is_scale=True, dropout=dropout)
        self.n_heads = n_heads
        self.kq_head_size = kq_size // n_heads
        self.value_head_size = kq_size // n_heads  # sic: reference attention.py:432
        self.kq_size = kq_size
        self.value_size = value_size
        self.out_size = out_size
        self.post_processor = (
            nn.Linear(value_size, out_size)
            if is_post_process or value_size != out_size
            else None
        )
        assert kq_size % n_heads == 0, f"{kq_size} % {n_heads} != 0"
        assert value_size % n_heads == 0, f"{value_size} % {n_heads} != 0"
        self.reset_parameters()

    def reset_parameters(self):
        weights_init(self)
        # init for the *effective* per-head fan-out (reference attention.py:449-455)
        std = math.sqrt(2.0 / (self.kq_size + self.kq_head_size))
        nn.init.normal_(self.key_transform.weight, mean=0, std=std)
        nn.init.normal_(self.query_transform.weight, mean=0, std=std)
        std = math.sqrt(2.0 / (self.value_size + self.value_head_size))
        nn.init.normal_(self.value_transform.weight, mean=0, std=std)

    def forward(self, keys, queries, values, rel_pos_enc=None, **kwargs):
        """keys [B,K,kq], queries [B,Q,kq], values [B,K,v] -> [B,Q,out]."""
        if (
            keys is queries
            and queries is values
            and not self.is_relative_pos
            and self.kq_size == self.value_size
        ):
            # self-attention: ONE GEMM for all three projections (the
            # weights are concatenated; only the query has a bias)
            w = torch.cat(
                [
                    self.key_transform.weight,
                    self.query_transform.weight,
                    self.value_transform.weight,
                ],
                dim=0,
            )
            proj = torch.nn.functional.linear(keys, w)
            keys, queries, values = proj.split(
                [self.kq_size, self.kq_size, self.value_size], dim=-1
            )
            if self.query_transform.bias is not None:
                queries = queries + self.query_transform.bias
        else:
            keys = self.key_transform(keys)
            queries = self.query_transform(queries)
            values = self.value_transform(values)

        queries = self._make_multiheaded(queries, self.kq_head_size)
        values = self._make_multiheaded(values, self.value_head_size)

        if self.is_relative_pos:
            # relative positions give every query its own key set
            batch_size, n_keys, kq_size = keys.shape
            n_queries = queries.size(1)
            keys = (keys.unsqueeze(1) + rel_pos_enc).view(
                batch_size, n_queries * n_keys, kq_size
            )
            keys = self._make_multiheaded(keys, self.kq_head_size)
            keys = keys.view(
                batch_size * self.n_heads, n_queries, n_keys, self.kq_head_size
            )
        else:
            keys = self._make_multiheaded(keys, self.kq_head_size)

        # [B*H, Q, head]
        context = self.dot(keys, queries, values)
        context = self._concatenate_multiheads(context, self.value_head_size)

        if self.post_processor is not None:
            context = self.post_processor(context)
        return context

    def _make_multiheaded(self, kvq, head_size):
        """[B, N, H*h] -> [H*B, N, h] (head-major batch stacking)."""
        batch_size = kvq.size(0)
        kvq = kvq.view(batch_size, -1, self.n_heads, head_size)
        return (
            kvq.permute(2, 0, 1, 3)
            .contiguous()
            .view(batch_size * self.n_heads, -1, head_size)
        )

    def _concatenate_multiheads(self, kvq, head_size):
        """Inverse of `_make_multiheaded`."""
        batch_size = kvq.size(0) // self.n_heads
        kvq = kvq.view(self.n_heads, batch_size, -1, head_size)
        return (
            kvq.permute(1, 2, 0, 3)
            .contiguous()
            .view(batch_size, -1, self.n_heads * head_size)
        )


@_register("transformer")
class TransformerAttender(MultiheadAttender):
    """Image-Transformer block: MHA + post-LN residual + FFN
    (reference attention.py:530-588)."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, is_post_process=False, **kwargs)
        assert self.kq_size == self.out_size
        self.layer_norm1 = nn.LayerNorm(self.out_size)
        self.layer_norm2 = nn.LayerNorm(self.out_size)
        self.mlp = MLP(
            self.out_size, self.out_size, hidden_size=self.out_size, activation=nn.ReLU()
        )
        self.reset_parameters()

    def _fused_block_ok(self, keys, queries, values):
        import os

        from npf.ops import has_extension

        return (
            keys.is_cuda
            and has_extension()
            and os.environ.get("NPF_FORCE_EAGER") != "1"
            and os.environ.get("NPF_NO_FUSED_ATTENDER") != "1"
            # bf16 block: engage only under autocast / bf16 inputs — fp32
            # training must keep fp32 numerics (the LL targets live in a
            # regime where bf16 rounding is irreducible noise)
            and (torch.is_autocast_enabled("cuda")
                 or keys.dtype == torch.bfloat16)
            and not self.is_relative_pos
            and self.kq_size == self.value_size == self.out_size
            and self.kq_size <= 128
            and self.kq_head_size == 16
            and isinstance(self.dot.dropout, nn.Identity)
            and keys.shape[-1] == self.kq_size
            and self.key_transform.weight.dtype == torch.float32
        )

    def forward(self, keys, queries, values, **kwargs):
        if self._fused_block_ok(keys, queries, values):
            return self._fused_forward(keys, queries, values)
        context = super().forward(keys, queries, values, **kwargs)
        context = self.layer_norm1(context + queries)
        context = self.layer_norm2(context + self.dot.dropout(self.mlp(context)))
        return context

    def _fused_forward(self, keys, queries, values):
        """5 kernels for the whole block (vs ~18 + casts composed):
        qkv-projection+head-split MFMA kernel -> fused attention ->
        add+LN1 (head merge folded into the gather) -> mlp_chain FFN ->
        add+LN2.  Numerics = autocast bf16 with fp32 statistics."""
        from npf.ops import attention_qkv
        from npf.ops.functional import add_layernorm, qkv_project_headsplit

        B, Qn, D = queries.shape
        Kn = keys.shape[1]
        if keys is queries and queries is values:
            (kh,) = qkv_project_headsplit(
                [keys], [self.key_transform.weight], [None], self.n_heads
            )
            qh, vh = qkv_project_headsplit(
                [queries, values],
                [self.query_transform.weight, self.value_transform.weight],
                [self.query_transform.bias, None],
                self.n_heads,
            )
        else:
            kh, qh, vh = qkv_project_headsplit(
                [keys, queries, values],
                [
                    self.key_transform.weight,
                    self.query_transform.weight,
                    self.value_transform.weight,
                ],
                [None, self.query_transform.bias, None],
                self.n_heads,
            )
        ctx_h = attention_qkv(kh, qh, vh)  # [H*B, Qn, 16]
        h1 = add_layernorm(
            ctx_h,
            queries,
            self.layer_norm1.weight,
            self.layer_norm1.bias,
            eps=self.layer_norm1.eps,
            headsplit=(B, Qn, self.n_heads),
        ).view(B, Qn, D)
        ffn = self.mlp(h1)  # mlp_chain fused on GPU
        out = add_layernorm(
            ffn.view(B, Qn, D),
            h1,
            self.layer_norm2.weight,
            self.layer_norm2.bias,
            eps=self.layer_norm2.eps,
        ).view(B, Qn, D)
        if not torch.is_autocast_enabled("cuda"):
            # outside autocast the caller's modules are fp32: hand back the
            # caller's dtype (under autocast bf16 flows on unchanged)
            out = out.to(queries.dtype)
        return out


@_register("differential")
class DifferentialAttender(nn.Module):
    """Multi-head differential attention: each head's map is the difference of
    two softmax maps, ``softmax(q1 k1^T) - lam softmax(q2 k2^T)``, so that what
    both maps give to every context point cancels.

    The weight is learned, ``lam = exp(lq1 . lk1) - exp(lq2 . lk2) + lam_init``
    with ``lam_init = 0.8 - 0.6 exp(-0.3 (depth - 1))``, and every head's result
    is normed by itself and scaled by ``1 - lam_init``, which leaves gradients
    the size that one map would give them.

    Parameters
    ----------
    n_heads : int
        Query heads; each holds two maps of ``kq_size / (2 n_heads)`` values.
    n_kv_heads : int, optional
        Key and value heads, shared by ``n_heads / n_kv_heads`` query heads
        each; `n_heads` by default.
    depth : int
        The layer's place in a stack, from 1; sets ``lam_init``.
    is_post_process : bool
        Linear map of the joined heads; needed where sizes differ.
    """

    def __init__(
        self,
        kq_size,
        value_size,
        out_size,
        n_heads=4,
        n_kv_heads=None,
        depth=1,
        is_post_process=True,
    ):
        super().__init__()
        n_kv_heads = n_heads if n_kv_heads is None else n_kv_heads
        if kq_size % (2 * n_heads):
            raise ValueError(f"kq_size {kq_size} is no multiple of {2 * n_heads}")
        if value_size % n_heads:
            raise ValueError(f"value_size {value_size} is no multiple of {n_heads}")
        if n_kv_heads < 1 or n_heads % n_kv_heads:
            raise ValueError(f"{n_heads} heads cannot share {n_kv_heads} key heads")
        if depth < 1:
            raise ValueError(f"depth starts at 1, got {depth}")
        self.kq_size = kq_size
        self.value_size = value_size
        self.out_size = out_size
        self.n_heads = n_heads
        self.n_kv_heads = n_kv_heads
        self.kq_head_size = kq_size // n_heads  # both maps
        self.value_head_size = value_size // n_heads
        self.lam_init = 0.8 - 0.6 * math.exp(-0.3 * (depth - 1))
        self.key_transform = nn.Linear(
            kq_size, n_kv_heads * self.kq_head_size, bias=False
        )
        self.query_transform = nn.Linear(kq_size, kq_size)
        self.value_transform = nn.Linear(
            value_size, n_kv_heads * self.value_head_size, bias=False
        )
        map_size = self.kq_head_size // 2
        self.lam_vectors = nn.Parameter(torch.empty(4, map_size))
        self.head_norm = nn.LayerNorm(self.value_head_size)
        self.post_processor = (
            nn.Linear(value_size, out_size)
            if is_post_process or value_size != out_size
            else None
        )
        self.reset_parameters()

    def reset_parameters(self):
        weights_init(self)
        nn.init.normal_(self.lam_vectors, std=0.1)

    def lam(self):
        """The weight of the second map, a 0-d fp32 tensor."""
        with torch.autocast(self.lam_vectors.device.type, enabled=False):
            lq1, lk1, lq2, lk2 = self.lam_vectors.float()
            return (lq1 * lk1).sum().exp() - (lq2 * lk2).sum().exp() + self.lam_init

    def forward(self, keys, queries, values, key_lengths=None):
        """keys [B,K,kq], queries [B,Q,kq], values [B,K,v] -> [B,Q,out].

        key_lengths: int [B], the valid contexts of each task; 0 is allowed.
        """
        B, Q, _ = queries.shape
        k = self._heads(self.key_transform(keys), self.n_kv_heads)
        q = self._heads(self.query_transform(queries), self.n_heads)
        v = self._heads(self.value_transform(values), self.n_kv_heads)
        context = ops.differential_attention(
            k, q, v, self.lam(), key_lengths=key_lengths
        )
        # [B, Q, H, Dv]: heads are joined by a view
        context = ops.layer_norm(
            context.transpose(1, 2),
            self.head_norm.weight,
            self.head_norm.bias,
            eps=self.head_norm.eps,
        ) * (1.0 - self.lam_init)
        context = context.reshape(B, Q, self.value_size)
        if self.post_processor is not None:
            context = self.post_processor(context)
        return context

    @staticmethod
    def _heads(x, n_heads):
        """[B, N, H*h] -> [B, H, N, h], a view."""
        # (the size is given: with no contexts it would not follow)
        return x.view(*x.shape[:2], n_heads, x.shape[-1] // n_heads).transpose(1, 2)


@_register("differential_transformer")
class DifferentialTransformerAttender(DifferentialAttender):
    """Differential attention with the transformer attender's block around it:
    residual and norm, then an MLP with residual and norm."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, is_post_process=False, **kwargs)
        if self.kq_size != self.out_size:
            raise ValueError(
                f"queries have size {self.kq_size}, the residual {self.out_size}"
            )
        self.layer_norm1 = nn.LayerNorm(self.out_size)
        self.layer_norm2 = nn.LayerNorm(self.out_size)
        self.mlp = MLP(
            self.out_size, self.out_size, hidden_size=self.out_size, activation=nn.ReLU()
        )
        self.reset_parameters()

    def forward(self, keys, queries, values, key_lengths=None):
        context = super().forward(keys, queries, values, key_lengths=key_lengths)
        context = self._add_norm(self.layer_norm1, context, queries)
        return self._add_norm(self.layer_norm2, self.mlp(context), context)

    @staticmethod
    def _add_norm(norm, x, residual):
        # under autocast the products are 16 bit and the residual may not be
        dtype = torch.promote_types(x.dtype, residual.dtype)
        return ops.layer_norm(
            x.to(dtype), norm.weight, norm.bias, eps=norm.eps,
            residual=residual.to(dtype),
        )
