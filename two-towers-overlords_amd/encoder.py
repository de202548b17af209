"""The frozen encoder of the `bert` mode on this package's own kernels, without padding.

    linear / attention / attention_qkv   differentiable forms of ops.linear_act and ops.packed_attention
    PackedBertEncoder                    a transformers BertModel's forward (what backend/model.py:51-52 executes) on tokens
                                         packed back to back: the texts of a batch have 10-130 tokens, the stock forward
                                         pads all of them to the longest

`AveragePoolingTower(encoder_impl="hip")` encodes through it (model.py); the default stays the stock PyTorch forward.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn.functional as F
from torch import Tensor, nn
from torch.autograd.function import once_differentiable

from . import ops

ACTIVATIONS = {"gelu": "gelu", "gelu_python": "gelu", "gelu_new": "gelu_tanh", "gelu_pytorch_tanh": "gelu_tanh", "gelu_fast": "gelu_tanh",
               "relu": "relu", "silu": "silu", "swish": "silu", "linear": "none"}


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, recording):
        need = recording and any(ctx.needs_input_grad[:3])  # (needs_input_grad is set under no_grad as well)
        y, z = ops.linear_act(x, weight, bias, residual, activation, save_preact=True) if need else (
            ops.linear_act(x, weight, bias, residual, activation), None)
        ctx.activation = activation
        ctx.save_for_backward(x, weight, z)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        nx, nw, nb, nr = ctx.needs_input_grad[:4]
        if dy.stride(-1) != 1 or (dy.shape[0] > 1 and dy.stride(0) < dy.shape[1]):
            dy = dy.contiguous()  # a broadcast upstream gradient (sum().backward())
        dx, dw, db = ops.linear_act_bwd(dy, x, weight, z, ctx.activation, bias=nb, need_dx=nx, need_dw=nw) if nx or nw or nb else (None,) * 3
        return dx, dw, db, dy if nr else None, None, None


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, residual: Optional[Tensor] = None, activation: str = "none") -> Tensor:
    """act(x @ weight.T + bias) + residual for x [..., K], residual [..., N]; differentiable in all four tensors."""
    lead = x.shape[:-1]
    if residual is not None:
        if residual.shape != lead + weight.shape[:1]:
            raise ValueError(f"residual: expected shape {tuple(lead + weight.shape[:1])}, got {tuple(residual.shape)}")
        residual = residual.reshape(-1, weight.shape[0])
    y = _LinearFn.apply(x.reshape(-1, x.shape[-1]), weight, bias, residual, activation, torch.is_grad_enabled())
    return y.view(*lead, weight.shape[0])


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, prefix, slopes, key_mask, kw):
        masks = dict(prefix=prefix, slopes=slopes, key_mask=key_mask)
        out, lse = ops.packed_attention(q, k, v, cu_seqlens, **masks, **kw)
        ctx.kw = kw
        ctx.save_for_backward(q, k, v, out, lse, cu_seqlens, prefix, slopes, key_mask)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, cu, prefix, slopes, key_mask = ctx.saved_tensors
        grads = ops.packed_attention_bwd(dout.contiguous(), q, k, v, out, lse, cu, prefix=prefix, slopes=slopes, key_mask=key_mask, **ctx.kw)
        return (*grads, None, None, None, None, None)


class _QkvAttentionFn(torch.autograd.Function):
    """q, k, v are column blocks of one projection's output, and so are their gradients: no concatenation."""

    @staticmethod
    def forward(ctx, qkv, heads, cu_seqlens, prefix, slopes, key_mask, kw):
        q, k, v = _blocks(qkv, heads)
        out, lse = ops.packed_attention(q, k, v, cu_seqlens, prefix=prefix, slopes=slopes, key_mask=key_mask, **kw)
        ctx.heads, ctx.kw = heads, kw
        ctx.save_for_backward(qkv, out, lse, cu_seqlens, prefix, slopes, key_mask)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        qkv, out, lse, cu, prefix, slopes, key_mask = ctx.saved_tensors
        grad = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        ops.packed_attention_bwd(dout.contiguous(), *_blocks(qkv, ctx.heads), out, lse, cu, prefix=prefix, slopes=slopes, key_mask=key_mask,
                                 **ctx.kw, grads=_blocks(grad, ctx.heads))
        return grad, None, None, None, None, None, None


def _blocks(qkv: Tensor, heads: int) -> Tuple[Tensor, Tensor, Tensor]:
    kv = (qkv.shape[1] - heads) // 2
    return qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]


def _refuse_bias_gradient(slopes: Optional[Tensor]) -> None:
    # here: inside an autograd function's forward no gradient is recorded, and ops.packed_attention's own check sees none asked for
    if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
        raise ValueError("slopes: the distance bias has no gradient")


def attention(q: Tensor, k: Tensor, v: Tensor, cu_seqlens: Tensor, *, scale: Optional[float] = None, causal: bool = False,
              prefix: Optional[Tensor] = None, softcap: float = 0.0, slopes: Optional[Tensor] = None,
              key_mask: Optional[Tensor] = None) -> Tensor:
    """`ops.packed_attention`, differentiable in q, k and v -> out [T, H, Dh]."""
    _refuse_bias_gradient(slopes)
    return _AttentionFn.apply(q, k, v, cu_seqlens, prefix, slopes, key_mask, dict(scale=scale, causal=causal, softcap=softcap))


def attention_qkv(qkv: Tensor, heads: int, cu_seqlens: Tensor, *, scale: Optional[float] = None, causal: bool = False,
                  prefix: Optional[Tensor] = None, softcap: float = 0.0, slopes: Optional[Tensor] = None,
                  key_mask: Optional[Tensor] = None) -> Tensor:
    """`attention` on one projection's output [T, heads + 2 kv_heads, Dh] (query heads first, then keys, then values)."""
    if qkv.dim() != 3 or qkv.shape[1] <= heads or (qkv.shape[1] - heads) % 2:
        raise ValueError(f"qkv: expected [tokens, heads + 2 kv_heads, head_dim] with {heads} query heads, got {tuple(qkv.shape)}")
    _refuse_bias_gradient(slopes)
    return _QkvAttentionFn.apply(qkv, heads, cu_seqlens, prefix, slopes, key_mask, dict(scale=scale, causal=causal, softcap=softcap))


class PackedBertEncoder:
    """A transformers `BertModel`'s forward on packed tokens.  Holds the module, not copies of its weights: loading a
    checkpoint, moving or fine-tuning it needs nothing here.  Under `torch.autocast` the products and the attention run in the
    autocast type, the residual sums and the norms in float32, like the stock forward's; else everything in the weights' own
    type.  Differentiable in the weights that require a gradient.  There is no dropout: a module in train mode whose dropout
    probabilities are not 0 is refused, unless `frozen` says that its weights are not trained — it then runs as in eval mode,
    which is what a feature cache of it holds."""

    def __init__(self, model: nn.Module, frozen: bool = False):
        cfg = getattr(model, "config", None)
        try:
            emb, layers = model.embeddings, list(model.encoder.layer)
            embeddings = [emb.word_embeddings, emb.position_embeddings, emb.token_type_embeddings]
            denses, norms = [], [emb.LayerNorm]
            for l in layers:
                at = l.attention
                denses += [at.self.query, at.self.key, at.self.value, at.output.dense, l.intermediate.dense, l.output.dense]
                norms += [at.output.LayerNorm, l.output.LayerNorm]
        except AttributeError as e:
            raise ValueError(f"encoder_impl='hip' runs BERT-shaped encoders only ({e})") from None
        # other families carry the same names and compute something else (RoBERTa counts positions from the padding id, ...)
        if getattr(cfg, "model_type", None) != "bert":
            raise ValueError(f"encoder_impl='hip' runs BERT-shaped encoders only (model_type {getattr(cfg, 'model_type', None)!r})")
        for part, kind in [*((p, nn.Embedding) for p in embeddings), *((p, nn.Linear) for p in denses), *((p, nn.LayerNorm) for p in norms)]:
            if getattr(type(part), "forward", None) is not kind.forward:  # an adapter or a quantised layer: its weight is not all of it
                raise ValueError(f"encoder_impl='hip' reads the weights of plain layers: {type(part).__name__} is not an nn.{kind.__name__}")
        act = getattr(cfg, "hidden_act", None)
        if act not in ACTIVATIONS:
            raise ValueError(f"encoder_impl='hip': hidden_act {act!r} is not one of {', '.join(ACTIVATIONS)}")
        if getattr(cfg, "position_embedding_type", "absolute") not in (None, "absolute") or getattr(cfg, "is_decoder", False):
            raise ValueError("encoder_impl='hip' runs bidirectional encoders with absolute positions only")
        self.heads = cfg.num_attention_heads
        self.head_dim = cfg.hidden_size // self.heads
        if self.head_dim * self.heads != cfg.hidden_size or not 8 <= self.head_dim <= 128 or self.head_dim % 8:
            raise ValueError(f"encoder_impl='hip': head size {cfg.hidden_size}/{self.heads} is not a multiple of 8 in 8..128")
        self.activation = ACTIVATIONS[act]
        self.model = model
        self.frozen = frozen

    @staticmethod
    def _types(weight: Tensor) -> Tuple[torch.dtype, torch.dtype]:
        """(type of the products, type of the rows between them)"""
        return (torch.get_autocast_dtype("cuda"), torch.float32) if torch.is_autocast_enabled("cuda") else (weight.dtype, weight.dtype)

    def __call__(self, input_ids: Tensor, attention_mask: Optional[Tensor] = None, token_type_ids: Optional[Tensor] = None):
        """input_ids [B, S] (padded, any mask pattern) -> (hidden [T, D] of the T attended tokens in row order, slots [T]: their
        places in the padded [B * S]).  One read-back: the number of attended tokens."""
        m = self.model
        if m.training and not self.frozen and any(isinstance(d, nn.Dropout) and d.p > 0 for d in m.modules()):
            raise RuntimeError("encoder_impl='hip' has no dropout: put the encoder in eval mode, or set its dropout probabilities to 0")
        B, S = input_ids.shape
        emb = m.embeddings
        if S > emb.position_embeddings.weight.shape[0]:
            raise ValueError(f"{S} tokens per text, the encoder has {emb.position_embeddings.weight.shape[0]} positions")
        dev = input_ids.device
        if attention_mask is None:
            slots = torch.arange(B * S, device=dev)
            lens = torch.full((B,), S, dtype=torch.int64, device=dev)
        else:
            keep = attention_mask != 0
            slots = keep.reshape(-1).nonzero().squeeze(1)
            lens = keep.sum(1)
        cu = F.pad(lens.cumsum(0), (1, 0)).to(torch.int32)
        dt, rows = self._types(emb.word_embeddings.weight)
        with torch.autocast("cuda", enabled=False):
            x = F.embedding(input_ids.reshape(-1)[slots].long(), emb.word_embeddings.weight, padding_idx=emb.word_embeddings.padding_idx)
            x = x + F.embedding(slots % S, emb.position_embeddings.weight)
            types = emb.token_type_embeddings.weight
            x = x + (types[0] if token_type_ids is None else F.embedding(token_type_ids.reshape(-1)[slots].long(), types))
            x = self._norm(x.to(rows), emb.LayerNorm)
            for layer in (m.encoder.layer if slots.numel() else ()):  # no token, nothing to do
                x = self._layer(x, cu, layer, dt)
        return x, slots

    @staticmethod
    def _norm(x: Tensor, ln: nn.LayerNorm) -> Tensor:
        return F.layer_norm(x, ln.normalized_shape, ln.weight.to(x.dtype), ln.bias.to(x.dtype), ln.eps)

    def _layer(self, x: Tensor, cu: Tensor, layer: nn.Module, dt: torch.dtype) -> Tensor:
        at = layer.attention
        qkv = (at.self.query, at.self.key, at.self.value)
        w = torch.cat([p.weight for p in qkv]).to(dt)
        b = torch.cat([p.bias for p in qkv]).to(dt)
        h = linear(x.to(dt), w, b).view(-1, 3 * self.heads, self.head_dim)
        h = attention_qkv(h, self.heads, cu).reshape(-1, self.heads * self.head_dim)
        x = self._norm(self._dense(h, at.output.dense, dt, residual=x), at.output.LayerNorm)
        h = self._dense(x.to(dt), layer.intermediate.dense, dt, activation=self.activation)
        return self._norm(self._dense(h, layer.output.dense, dt, residual=x), layer.output.LayerNorm)

    @staticmethod
    def _dense(x: Tensor, d: nn.Linear, dt: torch.dtype, residual: Optional[Tensor] = None, activation: str = "none") -> Tensor:
        fused = residual if residual is None or residual.dtype == dt else None
        y = linear(x, d.weight.to(dt), None if d.bias is None else d.bias.to(dt), fused, activation)
        return y if fused is residual else y + residual  # autocast: rows of float32

    def padded(self, input_ids: Tensor, attention_mask: Optional[Tensor] = None, token_type_ids: Optional[Tensor] = None) -> Tensor:
        """The stock forward's last_hidden_state [B, S, D] in float32, zero where a token is not attended."""
        B, S = input_ids.shape
        x, slots = self(input_ids, attention_mask, token_type_ids)
        out = torch.zeros(B * S, x.shape[1], dtype=torch.float32, device=x.device)
        return out.index_copy(0, slots, x.float()).view(B, S, x.shape[1])
