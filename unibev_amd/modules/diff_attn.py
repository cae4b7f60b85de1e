"""``DifferentialAttention`` — dense attention whose map is the difference of two softmax maps, for the self-attention slot of the
object-query decoder (beside ``MultiheadAttention``: same constructor keywords, call signature and masks).

A head of width Dv = embed_dims / num_heads scores with two query / key pairs of width Dv / 2:

    A = softmax(scale q_1 k_1^T + mask) - lam softmax(scale q_2 k_2^T + mask),   lam = exp(a_1 . b_1) - exp(a_2 . b_2) + lambda_init

(learned vectors a, b; one lam for the layer); the head's output A v is normalised by itself (weights shared by the heads) and
scaled by 1 - lambda_init before the output projection.  Attention, head-wise norm and residual dropout are this library's
kernels (``functional.diff_attention`` / ``layer_norm`` / ``dropout``); neither scores nor dropout masks are stored.
"""
import torch
import torch.nn as nn

from .. import functional as UF
from ..linear import linear as ubv_linear
from ..registry import ATTENTION
from .bricks import BaseModule, xavier_init


@ATTENTION.register_module()
class DifferentialAttention(BaseModule):
    """``num_kv_heads`` (default ``num_heads``) heads of keys and values are shared by groups of query heads; ``attn_drop`` drops
    entries of A; ``dropout`` sets attn_drop and the residual's dropout, as in ``MultiheadAttention``."""

    def __init__(self, embed_dims, num_heads, num_kv_heads=None, attn_drop=0., proj_drop=0.,
                 dropout_layer=dict(type='Dropout', drop_prob=0.), lambda_init=0.8, init_cfg=None, batch_first=False, **kwargs):
        super().__init__(init_cfg)
        if 'dropout' in kwargs:
            attn_drop = kwargs.pop('dropout')
            dropout_layer = dict(type='Dropout', drop_prob=attn_drop)
        num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        if embed_dims % (2 * num_heads):
            raise ValueError(f'embed_dims {embed_dims} must be a multiple of 2 * num_heads = {2 * num_heads}')
        if num_kv_heads < 1 or num_heads % num_kv_heads:
            raise ValueError(f'num_heads {num_heads} must be a multiple of num_kv_heads {num_kv_heads}')
        self.embed_dims, self.num_heads, self.num_kv_heads = embed_dims, num_heads, num_kv_heads
        self.head_dims = embed_dims // num_heads
        if self.head_dims > 256:
            raise ValueError(f'heads of width {self.head_dims} (at most 256)')
        self.batch_first = batch_first
        self.attn_drop, self.proj_drop = attn_drop, proj_drop
        self.residual_drop = (dropout_layer or {}).get('drop_prob', 0.)
        self.lambda_init = lambda_init
        self.q_proj = nn.Linear(embed_dims, embed_dims)
        self.k_proj = nn.Linear(embed_dims, num_kv_heads * self.head_dims)
        self.v_proj = nn.Linear(embed_dims, num_kv_heads * self.head_dims)
        self.out_proj = nn.Linear(embed_dims, embed_dims)
        self.lambda_a = nn.Parameter(torch.empty(2, self.head_dims // 2))
        self.lambda_b = nn.Parameter(torch.empty(2, self.head_dims // 2))
        self.head_norm = nn.LayerNorm(self.head_dims)
        self.init_weights()

    def init_weights(self):
        for m in (self.q_proj, self.k_proj, self.v_proj, self.out_proj):
            xavier_init(m, distribution='uniform')
        nn.init.normal_(self.lambda_a, std=0.1)
        nn.init.normal_(self.lambda_b, std=0.1)
        self._is_init = True

    def lam(self):
        """The layer's lam, (1,) f32."""
        e = (self.lambda_a.float() * self.lambda_b.float()).sum(-1).exp()
        return e[:1] - e[1:] + self.lambda_init

    def forward(self, query, key=None, value=None, identity=None, query_pos=None, key_pos=None, attn_mask=None,
                key_padding_mask=None, **kwargs):
        if key is None:
            key = query
        if value is None:
            value = key
        if identity is None:
            identity = query
        if key_pos is None and query_pos is not None and query_pos.shape == key.shape:
            key_pos = query_pos
        if query_pos is not None:
            query = query + query_pos
        if key_pos is not None:
            key = key + key_pos
        q, k, v = (ubv_linear(x, m.weight, m.bias) for x, m in ((query, self.q_proj), (key, self.k_proj), (value, self.v_proj)))
        if not self.batch_first:                               # (N, B, C): the operator takes the transposed views
            q, k, v = (t.transpose(0, 1) for t in (q, k, v))
        dv = self.head_dims
        o = UF.diff_attention(q.unflatten(-1, (self.num_heads, 2, dv // 2)), k.unflatten(-1, (self.num_kv_heads, 2, dv // 2)),
                              v.unflatten(-1, (self.num_kv_heads, dv)), self.lam(), attn_mask=attn_mask,
                              key_padding_mask=key_padding_mask, p=self.attn_drop, training=self.training)
        norm, keep = self.head_norm, 1.0 - self.lambda_init
        o = UF.layer_norm(o, norm.weight * keep, norm.bias * keep, norm.eps).flatten(-2)
        if not self.batch_first:
            o = o.transpose(0, 1)
        out = ubv_linear(o, self.out_proj.weight, self.out_proj.bias)
        out = UF.dropout(out, self.proj_drop, self.training)
        return UF.dropout(out, self.residual_drop, self.training, identity=identity)
