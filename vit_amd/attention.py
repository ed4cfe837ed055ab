"""Self-attention of the encoder block (reference: vit/attention.py:71-111,163-215,375-449).

``SelfAttention`` holds the same parameters under the same names as the reference; its forward unpacks them
into ``attention_qkv_packed``, which runs norm -> QKV GEMM -> RoPE -> flash attention -> out_proj GEMM as one
autograd function over libvitk kernels.  ``CrossAttention`` / ``AttentivePool`` (vit/attention.py:451-667) and the
``forward_weights`` diagnostics (vit/attention.py:281-373) run through ``ops.CrossAttentionFn`` and
``vitk_attn_weights``."""
from __future__ import annotations

import math
from typing import Any, NamedTuple, Optional, Union

import torch
import torch.nn as nn
from torch import Tensor

from . import kernels as K
from . import ops
from .initialization import init_linear, trunc_normal_
from .norm import get_norm_bias, is_layer_norm, make_norm
from .pos_enc import RelativeBuckets

_DTYPES = (torch.float32, torch.bfloat16)


def _heads(name: str, t: Tensor, like: Optional[Tensor] = None, head_dims: bool = True) -> None:
    if t.dim() != 4:
        raise ValueError(f"vit_amd: {name} must be [B, L, H, Dh], got {tuple(t.shape)}")
    if t.dtype not in _DTYPES:
        raise TypeError(f"vit_amd: {name} must be float32 or bfloat16, got {t.dtype}")
    if like is not None:
        if t.dtype != like.dtype:
            raise TypeError(f"vit_amd: {name} is {t.dtype}, the queries are {like.dtype}")
        if t.shape[0] != like.shape[0] or t.shape[3] != like.shape[3] or (head_dims and t.shape[2] != like.shape[2]):
            raise ValueError(f"vit_amd: {name} {tuple(t.shape)} does not go with the queries {tuple(like.shape)}")


def _key_counts(kv_lengths: Optional[Tensor], B: int) -> Optional[Tensor]:
    """int32 key counts [B]; values are clamped to [0, Lk] by the kernels (no value is read on the host)."""
    if kv_lengths is None:
        return None
    if not isinstance(kv_lengths, Tensor) or kv_lengths.dtype not in (torch.int32, torch.int64) or tuple(kv_lengths.shape) != (B,):
        raise ValueError(f"vit_amd: kv_lengths must be an int32 or int64 tensor of shape ({B},), got "
                         f"{(kv_lengths.dtype, tuple(kv_lengths.shape)) if isinstance(kv_lengths, Tensor) else type(kv_lengths)}")
    if kv_lengths.dtype == torch.int64:   # a count beyond 32 bits is as good as the largest one
        kv_lengths = kv_lengths.clamp(0, 2 ** 31 - 1).to(torch.int32)
    return kv_lengths.contiguous()


def _wants_grad(*ts: Optional[Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def qk_norm_rope(q: Tensor, k: Optional[Tensor], q_norm_weight: Tensor, k_norm_weight: Optional[Tensor] = None,
                 q_norm_bias: Optional[Tensor] = None, k_norm_bias: Optional[Tensor] = None, rope_q: Optional[Tensor] = None,
                 rope_k: Optional[Tensor] = None, *, eps: float = 1e-5, use_layer_norm: bool = False):
    """Per-head RMSNorm (or LayerNorm) of q [B, Lq, H, Dh] and k [B, Lk, Hk, Dh] followed by the position rotation, in one
    pass over both (vit/attention.py:25-41 and vit/rope.py:139-163); returns (q, k).  ``k`` may be None (a decoder step
    that rotates its query only).  Weights and biases are [Dh]; a table [2, N, Dh] or [2, B, 1, N, Dh] (sin, cos) rotates
    the last N rows.  Any strides with contiguous heads; head_dim a multiple of 8, at most 128; float32 or bfloat16.
    Arithmetic is float32, rounded once at the store.  Differentiable in q, k, the weights and the biases; the tables are
    constants, and one that asks for a gradient is refused."""
    _heads("q", q)
    Dh = q.shape[3]
    if k is not None:
        _heads("k", k, q, head_dims=False)
        if k_norm_weight is None:
            raise ValueError("vit_amd: k needs k_norm_weight")
    if not K.can_qk_norm_rope(q.dtype, Dh):
        raise ValueError(f"vit_amd: qk_norm_rope takes head sizes that are multiples of 8 up to 128, got {Dh}")
    if not eps >= 0.0:
        raise ValueError(f"vit_amd: eps must not be negative, got {eps}")
    wdt = q_norm_weight.dtype
    params = [q_norm_weight, k_norm_weight, q_norm_bias, k_norm_bias]
    for i, t in enumerate(params):
        if t is None:
            continue
        if t.shape != (Dh,) or t.dtype != wdt or wdt not in _DTYPES:
            name = ("q_norm_weight", "k_norm_weight", "q_norm_bias", "k_norm_bias")[i]
            raise ValueError(f"vit_amd: {name} must be [{Dh}] {wdt} (float32 or bfloat16), got {tuple(t.shape)} {t.dtype}")
        if not t.is_contiguous():
            params[i] = t.contiguous()
    q_norm_weight, k_norm_weight, q_norm_bias, k_norm_bias = params
    tables = []
    for name, x, rope in (("rope_q", q, rope_q), ("rope_k", k, rope_k)):
        if rope is None or x is None:
            tables.append(None)
            continue
        B, Ln = x.shape[0], x.shape[1]
        n = rope.shape[-2] if rope.dim() >= 2 else -1
        if (rope.shape != (2, n, Dh) and rope.shape != (2, B, 1, n, Dh)) or n > Ln:
            raise ValueError(f"vit_amd: {name} must be [2, N, {Dh}] or [2, {B}, 1, N, {Dh}] with N <= {Ln}, got {tuple(rope.shape)}")
        if _wants_grad(rope):
            raise ValueError(f"vit_amd: {name} is a constant table, its gradient is not computed; pass {name}.detach()")
        tables.append(rope if rope.dim() == 3 and rope.dtype == torch.float32 and rope.is_contiguous() and not rope.requires_grad
                      and not rope.data_ptr() & 15 else ops._rope_table(rope, None, B, B, q.dtype)[0])
    q, k = K.attn_operand(q), None if k is None else K.attn_operand(k)
    if _wants_grad(q, k, q_norm_weight, k_norm_weight, q_norm_bias, k_norm_bias):
        return ops.QkNormRopeFn.apply(q, k, q_norm_weight, k_norm_weight, q_norm_bias, k_norm_bias, *tables, float(eps),
                                      bool(use_layer_norm))
    qo = q.new_empty(q.shape)
    ko = None if k is None else k.new_empty(k.shape)
    K.qk_norm_rope_fwd(q, k, qo, ko, (q_norm_weight, k_norm_weight), (q_norm_bias, k_norm_bias), tables, float(eps),
                       bool(use_layer_norm), checked=True)
    return qo, ko


def attention(q: Tensor, k: Tensor, v: Tensor, *, bias_table: Optional[Tensor] = None, buckets: Optional[RelativeBuckets] = None,
              kv_lengths: Optional[Tensor] = None, scale: Optional[float] = None, dropout: float = 0.0,
              training: bool = False) -> Tensor:
    """softmax(scale q k^T + bias) v for q [B, Lq, H, Dh] and k, v [B, Lk, H, Dh]; returns [B, Lq, H, Dh].

    ``bias_table`` [num_buckets, H] with ``buckets`` (a ``RelativeBuckets`` of Lq x Lk pairs) adds a learned relative
    position bias to the scores; the table is used in the dtype of q and its gradient comes back in its own.
    ``kv_lengths`` [B] (int32 or int64) counts the keys each sample has; keys behind them are padding: never read, zero
    gradient.  A query that no key is left for gives zeros.  ``scale`` defaults to Dh ** -0.5.
    Any strides with contiguous heads, head_dim <= 128, float32 or bfloat16; Lq and Lk are independent, one query included.
    Head sizes that are no multiple of 8 run portable kernels, which take about a hundred times as long.  A bias needs memory
    while a call runs, per pair and head: 2 bytes in bfloat16, 4 in its backward, and 4 more (for each share of the samples, where
    their number is split to fill the chip) where the table's gradient is wanted, which float32 needs alone.
    Differentiable once in q, k, v and the table.  Tensors belong to the current device and stream."""
    _heads("q", q)
    _heads("k", k, q)
    _heads("v", v, q)
    if v.shape != k.shape:
        raise ValueError(f"vit_amd: k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    B, Lq, H, Dh = q.shape
    if Dh > 128 or Dh < 1:
        raise ValueError(f"vit_amd: head_dim must be in [1, 128], got {Dh}")
    if (bias_table is None) != (buckets is None):
        raise ValueError("vit_amd: a relative bias needs both bias_table and buckets")
    if buckets is not None:
        if buckets.shape != (Lq, k.shape[1]):
            raise ValueError(f"vit_amd: buckets cover {buckets.shape} pairs, the call has {(Lq, k.shape[1])}")
        if tuple(bias_table.shape) != (buckets.num_buckets, H) or bias_table.dtype not in _DTYPES:
            raise ValueError(f"vit_amd: bias_table must be [{buckets.num_buckets}, {H}] float32 or bfloat16, got "
                             f"{tuple(bias_table.shape)} {bias_table.dtype}")
    scale = Dh ** -0.5 if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"vit_amd: scale must be positive and finite, got {scale}")
    if not 0.0 <= dropout < 1.0:
        raise ValueError(f"vit_amd: dropout must be in [0, 1), got {dropout}")
    kv_len = _key_counts(kv_lengths, B)
    q, k, v = K.attn_operand(q), K.attn_operand(k), K.attn_operand(v)
    p = dropout if training else 0.0
    seed = ops.next_seed(q.device) if p > 0.0 else 0
    if _wants_grad(q, k, v, bias_table):
        return ops.AttentionFn.apply(q, k, v, bias_table, buckets, kv_len, scale, p, seed)
    if bias_table is not None:
        bias_table = bias_table.to(q.dtype).contiguous()
    return K.attn_var_fwd(q, k, v, table=bias_table, buckets=buckets, kv_len=kv_len, scale=scale, drop_p=p, seed=seed)[0]


def _sublayer_opts(*, head_dim, eps, layernorm, attention_dropout, dropout, training, residual, alpha=1.0,
                   qk_eps=1e-5, qk_layernorm=False):
    return dict(head_dim=head_dim, eps=float(eps), layernorm=bool(layernorm), attention_dropout=float(attention_dropout),
                dropout=float(dropout), training=bool(training), residual=residual, alpha=float(alpha),
                qk_eps=float(qk_eps), qk_layernorm=bool(qk_layernorm))


def attention_qkv_packed(x, w_in, b_in, w_norm, b_norm, use_layer_norm, head_dim, w_out, b_out, attn_mask, eps,
                         q_norm_weight, q_norm_bias, k_norm_weight, k_norm_bias, qk_use_layer_norm, qk_eps,
                         qk_normalization, attention_dropout, dropout, training, rope=None, *, bias_table=None,
                         buckets=None) -> Tensor:
    """Same positional signature as the reference function (vit/attention.py:164-189); returns the projected
    attention output (without the residual).  ``bias_table`` / ``buckets``: a learned relative position bias."""
    if attn_mask is not None:
        raise NotImplementedError("vit_amd: attention masks are not on the ViT encoder path (vit/transformer.py:151)")
    if qk_normalization:
        assert q_norm_weight is not None and k_norm_weight is not None
    else:
        q_norm_weight = q_norm_bias = k_norm_weight = k_norm_bias = None
    opt = _sublayer_opts(head_dim=head_dim, eps=eps, layernorm=use_layer_norm, attention_dropout=attention_dropout,
                         dropout=dropout, training=training, residual=False, qk_eps=qk_eps, qk_layernorm=qk_use_layer_norm)
    opt["buckets"] = buckets
    return ops.AttentionSublayerFn.apply(x, w_norm, b_norm, w_in, b_in, w_out, b_out, None, rope, None, q_norm_weight,
                                         q_norm_bias, k_norm_weight, k_norm_bias, opt, bias_table)


class SelfAttention(nn.Module):
    def __init__(self, hidden_size: int, num_attention_heads: int, hidden_dropout: float = 0.1,
                 attention_dropout: float = 0.1, bias: bool = True, eps: float = 1e-5,
                 qkv_quantization_config: Any = None, out_quantization_config: Any = None, device=None, dtype=None,
                 norm_type: str = "rmsnorm", qk_normalization: bool = False, relative_buckets: int = 0):
        super().__init__()
        if qkv_quantization_config is not None or out_quantization_config is not None:
            raise NotImplementedError("vit_amd: torchao quantization is outside the encoder hot path")
        kw = {"device": device, "dtype": dtype}
        self.norm = make_norm(hidden_size, norm_type, eps=eps, **kw)
        self._use_layer_norm = is_layer_norm(norm_type)
        # a learned relative position bias per head; the calls then name the bucket of every pair (RelativeBuckets)
        self.relative_bias = (nn.Parameter(torch.empty(relative_buckets, num_attention_heads, **kw)) if relative_buckets else None)
        self.qkv_proj = nn.Linear(hidden_size, 3 * hidden_size, bias=bias, **kw)
        self.out_proj = nn.Linear(hidden_size, hidden_size, bias=bias, **kw)
        self.dropout = nn.Dropout(hidden_dropout)
        self.attention_dropout = nn.Dropout(attention_dropout)
        self._head_dim = hidden_size // num_attention_heads
        self._qk_normalization = qk_normalization
        if qk_normalization:
            self.q_norm = make_norm(self._head_dim, norm_type, eps=eps, **kw)
            self.k_norm = make_norm(self._head_dim, norm_type, eps=eps, **kw)
        else:
            self.q_norm = self.k_norm = None
        self.reset_parameters()

    def reset_parameters(self) -> None:
        init_linear(self.qkv_proj)
        init_linear(self.out_proj)
        if self.relative_bias is not None:
            trunc_normal_(self.relative_bias)

    def _relative(self, buckets: Optional[RelativeBuckets], S: int):
        """(table, plan) of this call, (None, None) without a relative bias."""
        if (buckets is None) != (self.relative_bias is None):
            raise ValueError("vit_amd: a layer with a relative position bias is called with buckets, one without it is not")
        if buckets is not None and (buckets.shape != (S, S) or buckets.num_buckets != self.relative_bias.shape[0]):
            raise ValueError(f"vit_amd: buckets {buckets.shape} of {buckets.num_buckets} for a sequence of {S} and a table of "
                             f"{self.relative_bias.shape[0]}")
        return self.relative_bias, buckets

    def apply_quantization(self, qkv_quantization_config: Any = None, out_quantization_config: Any = None) -> None:
        if qkv_quantization_config is not None or out_quantization_config is not None:
            raise NotImplementedError("vit_amd: torchao quantization is outside the encoder hot path")

    def fused_residual(self, x: Tensor, rope: Optional[Tensor], gamma: Optional[Tensor], keep_idx: Optional[Tensor],
                       alpha: float, buckets: Optional[RelativeBuckets] = None) -> Tensor:
        """x (+) alpha * gamma * attention(x[keep_idx]) with residual, layer scale and drop-path merge fused."""
        table, buckets = self._relative(buckets, x.shape[1])
        qw, qb, kw_, kb, qk_eps = self._qk_norm_inputs()
        opt = _sublayer_opts(head_dim=self._head_dim, eps=self.norm.eps or 1e-5, layernorm=self._use_layer_norm,
                             attention_dropout=self.attention_dropout.p, dropout=self.dropout.p, training=self.training,
                             residual=True, alpha=alpha, qk_eps=qk_eps, qk_layernorm=self._use_layer_norm)
        opt["buckets"] = buckets
        return ops.AttentionSublayerFn.apply(x, self.norm.weight, get_norm_bias(self.norm), self.qkv_proj.weight,
                                             self.qkv_proj.bias, self.out_proj.weight, self.out_proj.bias, gamma, rope,
                                             keep_idx, qw, qb, kw_, kb, opt, table)

    def _qk_norm_inputs(self):
        """(q weight, q bias, k weight, k bias, eps), all None / 1e-5 without qk_normalization (vit/attention.py:61-68)."""
        if self.q_norm is None or self.k_norm is None:
            return None, None, None, None, 1e-5
        return (self.q_norm.weight, get_norm_bias(self.q_norm), self.k_norm.weight, get_norm_bias(self.k_norm),
                self.q_norm.eps or 1e-5)

    def forward_weights(self, x: Tensor, rope: Optional[Tensor] = None) -> Tensor:
        """Attention probabilities [B, H, S, S] (vit/attention.py:455-477)."""
        if self.relative_bias is not None:
            raise NotImplementedError("vit_amd: attention probabilities of a layer with a relative position bias")
        qw, qb, kw_, kb, qk_eps = self._qk_norm_inputs()
        opt = _sublayer_opts(head_dim=self._head_dim, eps=self.norm.eps or 1e-5, layernorm=self._use_layer_norm,
                             attention_dropout=0.0, dropout=0.0, training=False, residual=False, qk_eps=qk_eps,
                             qk_layernorm=self._use_layer_norm)
        return ops.self_attention_weights(x, self.norm.weight, get_norm_bias(self.norm), self.qkv_proj.weight,
                                          self.qkv_proj.bias, qw, qb, kw_, kb, rope, opt)

    def forward(self, x: Tensor, attn_mask: Optional[Tensor] = None, rope: Optional[Tensor] = None,
                buckets: Optional[RelativeBuckets] = None) -> Tensor:
        table, buckets = self._relative(buckets, x.shape[1])
        return attention_qkv_packed(
            x, self.qkv_proj.weight, self.qkv_proj.bias, self.norm.weight, get_norm_bias(self.norm), self._use_layer_norm,
            self._head_dim, self.out_proj.weight, self.out_proj.bias, attn_mask, self.norm.eps or 1e-5,
            *self._qk_norm_inputs()[:4], self._use_layer_norm, self._qk_norm_inputs()[4], self._qk_normalization,
            self.attention_dropout.p, self.dropout.p, self.training, rope, bias_table=table, buckets=buckets)


def attention_q_kv_packed(q, kv, w_q, b_q, w_kv, b_kv, w_norm, b_norm, use_layer_norm, head_dim, w_out, b_out, attn_mask,
                          eps, q_norm_weight, q_norm_bias, k_norm_weight, k_norm_bias, qk_use_layer_norm, qk_eps,
                          qk_normalization, attention_dropout, dropout, training, rope_q=None, rope_k=None, *,
                          kv_lengths=None) -> Tensor:
    """Same positional signature as the reference function (vit/attention.py:218-280).  ``kv_lengths`` [B]: the keys each
    sample of ``kv`` has; rows behind them are padding, whatever they hold: no output and no gradient depends on them."""
    if attn_mask is not None:
        raise NotImplementedError("vit_amd: attention masks are not built")
    if qk_normalization:
        assert q_norm_weight is not None and k_norm_weight is not None
    else:
        q_norm_weight = q_norm_bias = k_norm_weight = k_norm_bias = None
    opt = _sublayer_opts(head_dim=head_dim, eps=eps, layernorm=use_layer_norm, attention_dropout=attention_dropout,
                         dropout=dropout, training=training, residual=False, qk_eps=qk_eps, qk_layernorm=qk_use_layer_norm)
    opt["zero_padding"] = kv_lengths is not None and _wants_grad(kv, w_kv, b_kv, k_norm_weight, k_norm_bias)
    if opt["zero_padding"] and qk_normalization and not qk_eps > 0.0:
        raise ValueError("vit_amd: kv_lengths with head norms need qk_eps above 0 where gradients are taken (the norm of a padded row)")
    return ops.CrossAttentionFn.apply(q, kv, w_norm, b_norm, w_q, b_q, w_kv, b_kv, w_out, b_out, q_norm_weight, q_norm_bias,
                                      k_norm_weight, k_norm_bias, None, None, rope_q, rope_k, opt, _key_counts(kv_lengths, kv.shape[0]))


class KVMemory(NamedTuple):
    """Keys and values of a memory as ``CrossAttention.project_kv`` leaves them (normalised and rotated where the layer
    does that), for any number of forward calls without the projection."""

    kv: Tensor                      # [B, Lk, 2, H, Dh]: keys, values
    kv_lengths: Optional[Tensor]    # int32 [B] or None: all Lk keys


class CrossAttention(nn.Module):
    """Queries from one sequence, keys and values from another (vit/attention.py:480-592); pre-norm on the query side."""

    def __init__(self, hidden_size: int, num_attention_heads: int, hidden_dropout: float = 0.1,
                 attention_dropout: float = 0.1, bias: bool = True, eps: float = 1e-5,
                 qkv_quantization_config: Any = None, out_quantization_config: Any = None, device=None, dtype=None,
                 norm_type: str = "rmsnorm", qk_normalization: bool = False):
        super().__init__()
        if qkv_quantization_config is not None or out_quantization_config is not None:
            raise NotImplementedError("vit_amd: torchao quantization is outside the encoder hot path")
        kw = {"device": device, "dtype": dtype}
        self.norm = make_norm(hidden_size, norm_type, eps=eps, **kw)
        self._use_layer_norm = is_layer_norm(norm_type)
        self.q_proj = nn.Linear(hidden_size, hidden_size, bias=bias, **kw)
        self.kv_proj = nn.Linear(hidden_size, 2 * hidden_size, bias=bias, **kw)
        self.out_proj = nn.Linear(hidden_size, hidden_size, bias=bias, **kw)
        self.dropout = nn.Dropout(hidden_dropout)
        self.attention_dropout = nn.Dropout(attention_dropout)
        self._head_dim = hidden_size // num_attention_heads
        self._qk_normalization = qk_normalization
        if qk_normalization:
            self.q_norm = make_norm(self._head_dim, norm_type, eps=eps, **kw)
            self.k_norm = make_norm(self._head_dim, norm_type, eps=eps, **kw)
        else:
            self.q_norm = self.k_norm = None
        self.reset_parameters()

    def reset_parameters(self) -> None:
        init_linear(self.q_proj)
        init_linear(self.kv_proj)
        init_linear(self.out_proj)

    def apply_quantization(self, qkv_quantization_config: Any = None, out_quantization_config: Any = None) -> None:
        if qkv_quantization_config is not None or out_quantization_config is not None:
            raise NotImplementedError("vit_amd: torchao quantization is outside the encoder hot path")

    def _qk_norm_inputs(self):
        if self.q_norm is None or self.k_norm is None:
            return None, None, None, None, 1e-5
        return (self.q_norm.weight, get_norm_bias(self.q_norm), self.k_norm.weight, get_norm_bias(self.k_norm),
                self.q_norm.eps or 1e-5)

    def fused_residual(self, x: Tensor, kv: Tensor, gamma: Optional[Tensor], keep_idx: Optional[Tensor], alpha: float,
                       rope_q: Optional[Tensor] = None, rope_k: Optional[Tensor] = None,
                       kv_lengths: Optional[Tensor] = None) -> Tensor:
        """x (+) alpha * gamma * cross_attention(x[keep_idx], kv[keep_idx]): residual, layer scale and the drop-path merge
        in the out_proj epilogue (the cross sub-layer of vit/transformer.py:262-284)."""
        if isinstance(kv, KVMemory):
            if keep_idx is not None:
                raise ValueError("vit_amd: a projected memory is for inference; drop-path takes the memory's states")
            return self._from_memory(x, kv, gamma, rope_q, rope_k, kv_lengths, residual=True)
        qw, qb, kw_, kb, qk_eps = self._qk_norm_inputs()
        opt = _sublayer_opts(head_dim=self._head_dim, eps=self.norm.eps or 1e-5, layernorm=self._use_layer_norm,
                             attention_dropout=self.attention_dropout.p, dropout=self.dropout.p, training=self.training,
                             residual=True, alpha=alpha, qk_eps=qk_eps, qk_layernorm=self._use_layer_norm)
        opt["zero_padding"] = kv_lengths is not None and _wants_grad(kv, self.kv_proj.weight, self.kv_proj.bias, kw_, kb)
        return ops.CrossAttentionFn.apply(x, kv, self.norm.weight, get_norm_bias(self.norm), self.q_proj.weight,
                                          self.q_proj.bias, self.kv_proj.weight, self.kv_proj.bias, self.out_proj.weight,
                                          self.out_proj.bias, qw, qb, kw_, kb, gamma, keep_idx, rope_q, rope_k, opt,
                                          _key_counts(kv_lengths, kv.shape[0]))

    @torch.no_grad()
    def project_kv(self, kv: Tensor, rope_k: Optional[Tensor] = None, kv_lengths: Optional[Tensor] = None) -> KVMemory:
        """Keys and values of a memory [B, Lk, D], projected once: ``forward`` takes the result in place of the memory, so
        that a decoder's later steps (single tokens, mostly) read it and project nothing."""
        if kv.dim() != 3 or kv.shape[2] != self.kv_proj.in_features:
            raise ValueError(f"vit_amd: the memory must be [B, Lk, {self.kv_proj.in_features}], got {tuple(kv.shape)}")
        counts = _key_counts(kv_lengths, kv.shape[0])
        _, _, kw_, kb, qk_eps = self._qk_norm_inputs()
        packed = ops.project_memory(kv, self.kv_proj.weight, self.kv_proj.bias, kw_, kb, rope_k, self._head_dim, qk_eps,
                                    self._use_layer_norm)
        return KVMemory(packed, counts)

    def _from_memory(self, q: Tensor, memory: KVMemory, gamma: Optional[Tensor], rope_q, rope_k, kv_lengths, residual: bool):
        if rope_k is not None or kv_lengths is not None:
            raise ValueError("vit_amd: rope_k and kv_lengths of a projected memory are given to project_kv")
        if self.training or _wants_grad(q, *self.parameters()):
            raise RuntimeError("vit_amd: a projected memory is for inference: call eval() and use torch.no_grad()")
        B, Lq, D = q.shape
        H = D // self._head_dim
        if memory.kv.dim() != 5 or memory.kv.shape[0] != B or tuple(memory.kv.shape[2:]) != (2, H, self._head_dim):
            raise ValueError(f"vit_amd: memory {tuple(memory.kv.shape)} does not go with q {tuple(q.shape)}")
        qw, qb, _, _, qk_eps = self._qk_norm_inputs()
        return ops.cross_attention_from_memory(
            q, memory.kv, _key_counts(memory.kv_lengths, B), self.norm.weight, get_norm_bias(self.norm), self.norm.eps or 1e-5,
            self.q_proj.weight, self.q_proj.bias, self.out_proj.weight, self.out_proj.bias, qw, qb, qk_eps, self._use_layer_norm,
            rope_q, gamma, residual)

    def forward(self, q: Tensor, kv: Union[Tensor, KVMemory], attn_mask: Optional[Tensor] = None,
                rope_q: Optional[Tensor] = None, rope_k: Optional[Tensor] = None,
                kv_lengths: Optional[Tensor] = None) -> Tensor:
        if isinstance(kv, KVMemory):
            if attn_mask is not None:
                raise NotImplementedError("vit_amd: attention masks are not built")
            return self._from_memory(q, kv, None, rope_q, rope_k, kv_lengths, residual=False)
        qw, qb, kw_, kb, qk_eps = self._qk_norm_inputs()
        return attention_q_kv_packed(
            q, kv, self.q_proj.weight, self.q_proj.bias, self.kv_proj.weight, self.kv_proj.bias, self.norm.weight,
            get_norm_bias(self.norm), self._use_layer_norm, self._head_dim, self.out_proj.weight, self.out_proj.bias,
            attn_mask, self.norm.eps or 1e-5, qw, qb, kw_, kb, self._use_layer_norm, qk_eps, self._qk_normalization,
            self.attention_dropout.p, self.dropout.p, self.training, rope_q, rope_k, kv_lengths=kv_lengths)

    def forward_weights(self, q: Tensor, kv: Tensor, rope_q: Optional[Tensor] = None,
                        rope_k: Optional[Tensor] = None) -> Tensor:
        """Attention probabilities [B, H, Lq, Lk] (vit/attention.py:568-592)."""
        qw, qb, kw_, kb, qk_eps = self._qk_norm_inputs()
        opt = _sublayer_opts(head_dim=self._head_dim, eps=self.norm.eps or 1e-5, layernorm=self._use_layer_norm,
                             attention_dropout=0.0, dropout=0.0, training=False, residual=False, qk_eps=qk_eps,
                             qk_layernorm=self._use_layer_norm)
        return ops.cross_attention_weights(q, kv, self.norm.weight, get_norm_bias(self.norm), self.q_proj.weight,
                                           self.q_proj.bias, self.kv_proj.weight, self.kv_proj.bias, qw, qb, kw_, kb,
                                           rope_q, rope_k, opt)


class AttentivePool(nn.Module):
    """``num_queries`` learned queries attend over the tokens (vit/attention.py:594-667): [B, L, D] -> [B, D], or
    [B, num_queries, D] when there are several."""

    def __init__(self, hidden_size: int, num_attention_heads: int, num_queries: int = 1, hidden_dropout: float = 0.0,
                 attention_dropout: float = 0.0, bias: bool = True, device=None, dtype=None, norm_type: str = "rmsnorm",
                 qk_normalization: bool = False):
        super().__init__()
        if hidden_size % num_attention_heads != 0:
            raise ValueError(
                f"hidden_size ({hidden_size}) must be divisible by num_attention_heads ({num_attention_heads})")
        if num_queries < 1:
            raise ValueError(f"num_queries must be positive, got {num_queries}")
        self.query = nn.Parameter(torch.empty(1, num_queries, hidden_size, device=device, dtype=dtype))
        self.cross_attention = CrossAttention(hidden_size, num_attention_heads, hidden_dropout=hidden_dropout,
                                              attention_dropout=attention_dropout, bias=bias, device=device, dtype=dtype,
                                              norm_type=norm_type, qk_normalization=qk_normalization)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        trunc_normal_(self.query)
        self.cross_attention.reset_parameters()

    def forward(self, x: Tensor, lengths: Optional[Tensor] = None) -> Tensor:
        """``lengths`` [B]: the tokens each sample has; rows of x behind them are padding, whatever they hold."""
        y = self.cross_attention(self.query.expand(x.shape[0], -1, -1), x, kv_lengths=lengths)
        return y.squeeze(1) if y.shape[1] == 1 else y

    def forward_weights(self, x: Tensor) -> Tensor:
        """[B, H, num_queries, L] (vit/attention.py:658-659)."""
        return self.cross_attention.forward_weights(self.query.expand(x.shape[0], -1, -1), x)
