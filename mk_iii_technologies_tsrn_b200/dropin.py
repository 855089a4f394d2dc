"""Drop-in tropical transformer layers and models (tropformer_dropin.py).

Mirrors the public classes of tropformer_dropin.py -- same constructors,
parameter names and state-dict keys, PyTorch-style ``forward`` signatures --
with the tropical parts on this library's kernels:

* ``TropicalLinear`` (tropformer_dropin.py:45-79): the max-plus GEMM, STE
  backward in training, argmax backward in eval (the class of tropical.py;
  the math of both reference files is the same);
* the tropical attention score ``max_f(Q + K) * d_k^-1/2`` of
  ``TropicalMultiHeadAttention`` (:167-285, score at :236-240): the batched
  strided max-plus kernel over the [B, H, L, d_k] head views, with the argmax
  scatter backward that autograd of ``.max(-1)`` gives (value-only kernel
  when no gradient is taken), also across a ``TropicalKVCache``;
* ``TropicalHybridFFN`` (:288-328): in inference ``lf_act(trop_up(x))`` is one
  kernel (the LF activation fused into the max-plus epilogue);
* the scaled token embedding with learned positions of the token models
  (:616-720): one kernel, its gradient by sorted tokens (``ops.embedding``; the
  values are those of the PyTorch expression bit for bit).  An id outside the
  table makes its rows NaN, and a later call of the model raises
  ``ops.DeviceIndexError``, where PyTorch's embedding ends the CUDA context;
* decoding: ``TropicalDecoderModel.generate`` keeps keys and values in pages
  (``TropicalPagedKVCache``), each token's attention is one kernel over them
  (``ops.paged_attention``), the next token one more (``ops.sample_tokens``),
  and a budget of slots evicts by accumulated attention weight
  (``ops.cache_evict``).  The reference has no decoding loop; its concatenated
  ``TropicalKVCache`` stays as it is.

Everything else (projections, gate, masks, Maslov softmax, layer norms,
residuals) is the reference's PyTorch expression.  The encoder /
decoder layers, stacks and models below only compose these, as the reference
ones do; alternatively swap ``TropicalLinear``, ``TropicalMultiHeadAttention``
and ``TropicalHybridFFN`` into the reference module before building a model.
"""
from __future__ import annotations

import copy
import math
from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd import forward_ad
from torch.nn.modules import module as _module

from . import ops
from . import tropical
from .tropical import MaslovTemperature, TropicalLinear

__all__ = [
    "TropicalLinear", "MaslovTemperature", "LFDualActivation", "TropicalKVCache",
    "TropicalPagedKVCache", "TropicalMultiHeadAttention", "TropicalHybridFFN", "TropicalEncoderLayer",
    "TropicalDecoderLayer", "TropicalEncoder", "TropicalDecoder", "TropicalTransformer",
    "TropicalEncoderModel", "TropicalDecoderModel", "TropicalViT",
    "TropicalViTForClassification", "make_causal_mask", "maslov_summary", "lf_blend_summary",
]


class LFDualActivation(tropical.LFDualActivation):
    """Tropical polynomial activation and its Legendre-Fenchel dual
    (tropformer_dropin.py:100-140); "blend" is this file's default mode."""

    def __init__(self, dim: int, num_pieces: int = 8, mode: str = "blend"):
        super().__init__(dim, num_pieces=num_pieces, mode=mode)


@dataclass
class TropicalKVCache:
    """Keys and values of earlier decoding steps (tropformer_dropin.py:143-164);
    new ones are appended along the sequence axis (dim 2 of [B, H, L, d_k])."""

    k: Optional[torch.Tensor] = None
    v: Optional[torch.Tensor] = None

    def update(self, k_new: torch.Tensor, v_new: torch.Tensor):
        if self.k is None:
            self.k, self.v = k_new, v_new
        else:
            self.k = torch.cat([self.k, k_new], dim=2)
            self.v = torch.cat([self.v, v_new], dim=2)
        return self.k, self.v

    def reset(self):
        self.k = self.v = None


class TropicalPagedKVCache:
    """Keys and values of a model's layers in pages, for decoding (no reference counterpart; the
    single-layer :class:`TropicalKVCache` copies all of a cache for every token).

    ``num_layers`` pairs of [pages, page_size, num_heads, head_dim] tensors with room for
    ``max_slots`` slots of each of ``batch`` sequences, one ``block_table`` and one ``lengths`` for
    all layers.  A model's attention modules get ``cache.layer(i)`` as their ``cache``: between
    :meth:`begin` and the first :meth:`step` they attend over the prompt as without a cache and
    store it, after a :meth:`step` over the slots.  ``collect_mass`` sums the attention weights
    that :meth:`evict` goes by.  Inference only."""

    def __init__(self, num_layers: int, batch: int, num_heads: int, head_dim: int, max_slots: int,
                 *, page_size: int = 16, collect_mass: bool = False,
                 dtype: torch.dtype = torch.float32, device=None):
        per = -(-max_slots // page_size)
        shape = (batch * per, page_size, num_heads, head_dim)
        self.max_slots, self.most, self.prompting = max_slots, 0, False
        self.k = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        self.block_table = torch.arange(batch * per, dtype=torch.int32,
                                        device=device).view(batch, per)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.mass = [torch.zeros(batch, num_heads, per * page_size, device=device)
                     for _ in range(num_layers)] if collect_mass else [None] * num_layers

    def layer(self, i: int) -> "_PagedLayer":
        return _PagedLayer(self, i)

    def _room(self, slots: int) -> None:
        if slots > self.max_slots:
            raise ValueError(f"{slots} slots do not fit a cache of {self.max_slots}")
        self.most = slots

    def begin(self, counts: torch.Tensor, width: int) -> None:
        """A prompt of ``counts`` [batch] tokens (of ``width`` at most) follows."""
        self._room(width)
        self.prompting = True
        self.lengths.copy_(counts)

    def step(self) -> None:
        """One more token of every sequence follows."""
        self._room(self.most + 1)
        self.prompting = False
        self.lengths.add_(1)

    def evict(self, keep: int, recent: int = 0) -> None:
        """Leaves ``keep`` slots of each sequence (``ops.cache_evict``, every layer and head by its
        own weights)."""
        if self.mass[0] is None:
            raise ValueError("eviction needs collect_mass=True")
        for k, v, mass in zip(self.k, self.v, self.mass):
            ops.cache_evict(k, v, self.block_table, self.lengths, mass, keep, recent)
        self.lengths.clamp_(max=keep)
        self.most = min(self.most, keep)


@dataclass
class _PagedLayer:
    cache: TropicalPagedKVCache
    index: int

    def store(self, K: torch.Tensor, V: torch.Tensor, attn: torch.Tensor) -> None:
        # a prompt's keys and values [B, H, L, d_k] and softmax weights [B, H, L, L]
        c, i = self.cache, self.index
        ops.paged_append(K.transpose(1, 2), V.transpose(1, 2), c.k[i], c.v[i], c.block_table,
                         torch.zeros_like(c.lengths), c.lengths)
        if c.mass[i] is not None:
            L = attn.shape[-1]
            there = torch.arange(L, device=attn.device) < c.lengths[:, None]
            c.mass[i][:, :, :L] = (attn.float() * there[:, None, :, None]).sum(2)

    def attend(self, Q, K, V, scale, gate, tau):
        # Q, K, V [B, H, 1, d_k] of the new token (under autocast the gate is of their type)
        c, i = self.cache, self.index
        return ops.paged_attention(Q[:, :, 0], c.k[i], c.v[i], c.block_table, c.lengths,
                                   key=K[:, :, 0], value=V[:, :, 0], scale=scale,
                                   gate=gate.float(), tau=tau.float(), mass=c.mass[i])


def _grad_needed(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class TropicalMultiHeadAttention(nn.Module):
    """Self- or cross-attention blending tropical and classical scores
    (tropformer_dropin.py:167-285): ``g * trop + (1 - g) * classical`` with a
    sigmoid gate from the queries (cross: from the mean query and key
    contexts), additive and padding masks, Maslov softmax, @V, out_proj."""

    def __init__(self, d_model: int, num_heads: int, dropout: float = 0.1,
                 init_temp: float = 1.0, is_cross_attention: bool = False):
        super().__init__()
        assert d_model % num_heads == 0
        self.d_model = d_model
        self.num_heads = num_heads
        self.d_k = d_model // num_heads
        self._scale = self.d_k ** -0.5
        self.is_cross_attention = is_cross_attention
        self.q_proj = nn.Linear(d_model, d_model)
        self.k_proj = nn.Linear(d_model, d_model)
        self.v_proj = nn.Linear(d_model, d_model)
        self.out_proj = nn.Linear(d_model, d_model)
        self.score_gate = nn.Linear((2 if is_cross_attention else 1) * d_model, num_heads)
        nn.init.zeros_(self.score_gate.weight)
        nn.init.constant_(self.score_gate.bias, -2.0)
        self.maslov = MaslovTemperature(num_heads, init_temp)
        self.attn_dropout = nn.Dropout(dropout)

    def _split_heads(self, x: torch.Tensor) -> torch.Tensor:
        B, L, _ = x.shape
        return x.view(B, L, self.num_heads, self.d_k).transpose(1, 2)

    def _tropical_scores(self, Q: torch.Tensor, K: torch.Tensor) -> torch.Tensor:
        if _grad_needed(Q, K):
            return ops.TropicalScoreFunction.apply(Q, K, self._scale, None)
        return ops.tropical_scores(Q, K, self._scale, argmax=False)[0]

    def forward(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                attn_mask: Optional[torch.Tensor] = None,
                key_padding_mask: Optional[torch.Tensor] = None,
                cache: Optional[TropicalKVCache] = None, need_weights: bool = False):
        B, L_q, D = query.shape
        Q = self._split_heads(self.q_proj(query))
        K = self._split_heads(self.k_proj(key))
        V = self._split_heads(self.v_proj(value))
        paged = cache if isinstance(cache, _PagedLayer) else None
        if paged is not None:
            if self.is_cross_attention or (self.training and self.attn_dropout.p > 0):
                raise RuntimeError("a paged cache serves self-attention without dropout")
            if not paged.cache.prompting:
                if L_q != 1 or need_weights or attn_mask is not None or \
                        key_padding_mask is not None:
                    raise ValueError("after a prompt a paged cache takes one token at a time, "
                                     "without masks or weights")
                gate = torch.sigmoid(self.score_gate(query))[:, 0]                # (B, H)
                out = paged.attend(Q, K, V, self._scale, gate, self.maslov.temperatures)
                return self.out_proj(out.reshape(B, 1, D)), None
        elif cache is not None:
            K, V = cache.update(K, V)
        class_scores = torch.matmul(Q, K.transpose(-2, -1)) * self._scale
        trop_scores = self._tropical_scores(Q, K)
        if self.is_cross_attention:
            ctx = torch.cat([query.mean(dim=1), key.mean(dim=1)], dim=-1)
            g = torch.sigmoid(self.score_gate(ctx))[:, :, None, None]          # (B, H, 1, 1)
        else:
            g = torch.sigmoid(self.score_gate(query)).permute(0, 2, 1)[..., None]  # (B, H, Lq, 1)
        scores = g * trop_scores + (1.0 - g) * class_scores
        if attn_mask is not None:
            if attn_mask.dim() == 2:
                scores = scores + attn_mask[None, None]
            elif attn_mask.dim() == 3:
                scores = scores + attn_mask[:, None]
            else:
                scores = scores + attn_mask
        if key_padding_mask is not None:
            scores = scores.masked_fill(key_padding_mask[:, None, None, :], -1e9)
        attn = self.attn_dropout(self.maslov(scores))
        if paged is not None:
            paged.store(K, V, attn)
        out = torch.matmul(attn, V).transpose(1, 2).contiguous().view(B, L_q, D)
        return self.out_proj(out), (attn if need_weights else None)


class TropicalHybridFFN(nn.Module):
    """Tropical branch (TropicalLinear -> LFDualActivation -> dropout) and
    classical branch (Linear -> GELU) fused by sigmoid(gate_proj(x)), then
    down_proj and dropout (tropformer_dropin.py:288-328; no norm or residual)."""

    def __init__(self, d_model: int, ffn_dim: int, dropout: float = 0.1,
                 lf_pieces: int = 8, lf_mode: str = "blend"):
        super().__init__()
        self.trop_up = TropicalLinear(d_model, ffn_dim)
        self.lf_act = LFDualActivation(ffn_dim, num_pieces=lf_pieces, mode=lf_mode)
        self.trop_drop = nn.Dropout(dropout)
        self.class_up = nn.Linear(d_model, ffn_dim)
        self.gelu = nn.GELU()
        self.gate_proj = nn.Linear(d_model, ffn_dim)
        nn.init.zeros_(self.gate_proj.weight)
        nn.init.constant_(self.gate_proj.bias, -2.0)
        self.down_proj = nn.Linear(ffn_dim, d_model)
        self.dropout = nn.Dropout(dropout)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        trop = self.trop_drop(tropical.tropical_up_lf(self.trop_up, self.lf_act, x))
        classical = self.gelu(self.class_up(x))
        g = torch.sigmoid(self.gate_proj(x))
        return self.dropout(self.down_proj(g * trop + (1.0 - g) * classical))


class TropicalEncoderLayer(nn.Module):
    """Drop-in for nn.TransformerEncoderLayer (tropformer_dropin.py:331-403):
    forward(src, src_mask=None, src_key_padding_mask=None); pre-norm by default."""

    def __init__(self, d_model: int, nhead: int, dim_feedforward: int = 2048,
                 dropout: float = 0.1, lf_pieces: int = 8, lf_mode: str = "blend",
                 init_temp: float = 1.0, batch_first: bool = True, norm_first: bool = True):
        super().__init__()
        self.batch_first = batch_first
        self.norm_first = norm_first
        self.self_attn = TropicalMultiHeadAttention(d_model, nhead, dropout=dropout,
                                                    init_temp=init_temp)
        self.ffn = TropicalHybridFFN(d_model, dim_feedforward, dropout=dropout,
                                     lf_pieces=lf_pieces, lf_mode=lf_mode)
        self.norm1 = nn.LayerNorm(d_model)
        self.norm2 = nn.LayerNorm(d_model)
        self.dropout1 = nn.Dropout(dropout)
        self.dropout2 = nn.Dropout(dropout)

    def forward(self, src: torch.Tensor, src_mask: Optional[torch.Tensor] = None,
                src_key_padding_mask: Optional[torch.Tensor] = None,
                cache: Optional[TropicalKVCache] = None) -> torch.Tensor:
        x = src if self.batch_first else src.transpose(0, 1)
        masks = dict(attn_mask=src_mask, key_padding_mask=src_key_padding_mask)
        if cache is not None:           # (an attention of another make need not know of it)
            masks["cache"] = cache
        if self.norm_first:
            h = self.norm1(x)
            x = x + self.dropout1(self.self_attn(h, h, h, **masks)[0])
            x = x + self.dropout2(self.ffn(self.norm2(x)))
        else:
            x = self.norm1(x + self.dropout1(self.self_attn(x, x, x, **masks)[0]))
            x = self.norm2(x + self.dropout2(self.ffn(x)))
        return x if self.batch_first else x.transpose(0, 1)


class TropicalDecoderLayer(nn.Module):
    """Drop-in for nn.TransformerDecoderLayer (tropformer_dropin.py:406-492):
    self-attention, cross-attention over ``memory``, hybrid FFN."""

    def __init__(self, d_model: int, nhead: int, dim_feedforward: int = 2048,
                 dropout: float = 0.1, lf_pieces: int = 8, lf_mode: str = "blend",
                 init_temp: float = 1.0, batch_first: bool = True, norm_first: bool = True):
        super().__init__()
        self.batch_first = batch_first
        self.norm_first = norm_first
        self.self_attn = TropicalMultiHeadAttention(d_model, nhead, dropout=dropout,
                                                    init_temp=init_temp)
        self.cross_attn = TropicalMultiHeadAttention(d_model, nhead, dropout=dropout,
                                                     init_temp=init_temp, is_cross_attention=True)
        self.ffn = TropicalHybridFFN(d_model, dim_feedforward, dropout=dropout,
                                     lf_pieces=lf_pieces, lf_mode=lf_mode)
        self.norm1 = nn.LayerNorm(d_model)
        self.norm2 = nn.LayerNorm(d_model)
        self.norm3 = nn.LayerNorm(d_model)
        self.dropout1 = nn.Dropout(dropout)
        self.dropout2 = nn.Dropout(dropout)
        self.dropout3 = nn.Dropout(dropout)

    def forward(self, tgt: torch.Tensor, memory: torch.Tensor,
                tgt_mask: Optional[torch.Tensor] = None,
                memory_mask: Optional[torch.Tensor] = None,
                tgt_key_padding_mask: Optional[torch.Tensor] = None,
                memory_key_padding_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        if not self.batch_first:
            tgt, memory = tgt.transpose(0, 1), memory.transpose(0, 1)
        x = tgt
        self_masks = dict(attn_mask=tgt_mask, key_padding_mask=tgt_key_padding_mask)
        mem_masks = dict(attn_mask=memory_mask, key_padding_mask=memory_key_padding_mask)
        if self.norm_first:
            h = self.norm1(x)
            x = x + self.dropout1(self.self_attn(h, h, h, **self_masks)[0])
            h = self.norm2(x)
            x = x + self.dropout2(self.cross_attn(h, memory, memory, **mem_masks)[0])
            x = x + self.dropout3(self.ffn(self.norm3(x)))
        else:
            x = self.norm1(x + self.dropout1(self.self_attn(x, x, x, **self_masks)[0]))
            x = self.norm2(x + self.dropout2(self.cross_attn(x, memory, memory, **mem_masks)[0]))
            x = self.norm3(x + self.dropout3(self.ffn(x)))
        return x if self.batch_first else x.transpose(0, 1)


class TropicalEncoder(nn.Module):
    """Stack of copies of an encoder layer, optional final norm
    (tropformer_dropin.py:495-515).  ``cache``: a :class:`TropicalPagedKVCache`, whose layers go to
    the stack's in turn."""

    def __init__(self, encoder_layer: TropicalEncoderLayer, num_layers: int,
                 norm: Optional[nn.Module] = None):
        super().__init__()
        self.layers = nn.ModuleList([copy.deepcopy(encoder_layer) for _ in range(num_layers)])
        self.norm = norm

    def forward(self, src: torch.Tensor, mask: Optional[torch.Tensor] = None,
                src_key_padding_mask: Optional[torch.Tensor] = None,
                cache: Optional[TropicalPagedKVCache] = None) -> torch.Tensor:
        out = src
        for i, layer in enumerate(self.layers):
            cached = {} if cache is None else {"cache": cache.layer(i)}
            out = layer(out, src_mask=mask, src_key_padding_mask=src_key_padding_mask, **cached)
        return self.norm(out) if self.norm is not None else out


class TropicalDecoder(nn.Module):
    """Stack of copies of a decoder layer, optional final norm
    (tropformer_dropin.py:518-546)."""

    def __init__(self, decoder_layer: TropicalDecoderLayer, num_layers: int,
                 norm: Optional[nn.Module] = None):
        super().__init__()
        self.layers = nn.ModuleList([copy.deepcopy(decoder_layer) for _ in range(num_layers)])
        self.norm = norm

    def forward(self, tgt: torch.Tensor, memory: torch.Tensor,
                tgt_mask: Optional[torch.Tensor] = None,
                memory_mask: Optional[torch.Tensor] = None,
                tgt_key_padding_mask: Optional[torch.Tensor] = None,
                memory_key_padding_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        out = tgt
        for layer in self.layers:
            out = layer(out, memory, tgt_mask=tgt_mask, memory_mask=memory_mask,
                        tgt_key_padding_mask=tgt_key_padding_mask,
                        memory_key_padding_mask=memory_key_padding_mask)
        return self.norm(out) if self.norm is not None else out


class TropicalTransformer(nn.Module):
    """Encoder-decoder drop-in for nn.Transformer (tropformer_dropin.py:549-613)."""

    def __init__(self, d_model: int = 512, nhead: int = 8, num_encoder_layers: int = 6,
                 num_decoder_layers: int = 6, dim_feedforward: int = 2048, dropout: float = 0.1,
                 lf_pieces: int = 8, lf_mode: str = "blend", init_temp: float = 1.0,
                 batch_first: bool = True, norm_first: bool = True):
        super().__init__()
        args = (d_model, nhead, dim_feedforward, dropout, lf_pieces, lf_mode, init_temp,
                batch_first, norm_first)
        self.encoder = TropicalEncoder(TropicalEncoderLayer(*args), num_encoder_layers,
                                       norm=nn.LayerNorm(d_model) if norm_first else None)
        self.decoder = TropicalDecoder(TropicalDecoderLayer(*args), num_decoder_layers,
                                       norm=nn.LayerNorm(d_model) if norm_first else None)
        self.d_model = d_model
        self.nhead = nhead
        self.batch_first = batch_first

    def forward(self, src: torch.Tensor, tgt: torch.Tensor,
                src_mask: Optional[torch.Tensor] = None, tgt_mask: Optional[torch.Tensor] = None,
                memory_mask: Optional[torch.Tensor] = None,
                src_key_padding_mask: Optional[torch.Tensor] = None,
                tgt_key_padding_mask: Optional[torch.Tensor] = None,
                memory_key_padding_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        memory = self.encoder(src, mask=src_mask, src_key_padding_mask=src_key_padding_mask)
        return self.decoder(tgt, memory, tgt_mask=tgt_mask, memory_mask=memory_mask,
                            tgt_key_padding_mask=tgt_key_padding_mask,
                            memory_key_padding_mask=memory_key_padding_mask)


def make_causal_mask(seq_len: int, device: torch.device) -> torch.Tensor:
    """Additive causal mask, -1e9 above the diagonal (tropformer_dropin.py:723-733;
    a finite tropical zero keeps the max-plus score free of -inf)."""
    return torch.triu(torch.full((seq_len, seq_len), -1e9, device=device), diagonal=1)


def _plain_table(m: nn.Module) -> bool:
    # an nn.Embedding that is only its float32 table: no hooks, own forward, parametrisation,
    # renormalisation or other gradient than the dense sum
    return (type(m) is nn.Embedding and type(m.weight) in (nn.Parameter, torch.Tensor)
            and m.weight.dtype == torch.float32 and m.weight.is_cuda and m.max_norm is None
            and not m.sparse and not m.scale_grad_by_freq and not m._forward_hooks
            and not m._forward_pre_hooks and not m._backward_hooks and not m._backward_pre_hooks
            and "forward" not in m.__dict__)


def _global_hooks() -> bool:
    # hooks on every module (module trackers, counters): they want the modules themselves run
    return bool(_module._global_forward_hooks or _module._global_forward_pre_hooks
                or _module._global_backward_hooks or _module._global_backward_pre_hooks)


def _transformed(t: torch.Tensor) -> bool:
    # carries the tangent of a forward-mode derivative, or a wrapper of torch.func
    return (forward_ad.unpack_dual(t).tangent is not None
            or torch._C._functorch.is_functorch_wrapped_tensor(t))


class _TokenModel(nn.Module):
    # token + learned position embeddings scaled by sqrt(d_model), then an
    # encoder stack with a final norm (the shared body of the two models below)
    def _body(self, vocab_size, d_model, nhead, num_layers, dim_feedforward, dropout,
              max_seq_len, lf_pieces, lf_mode, init_temp):
        self.d_model = d_model
        self.embed = nn.Embedding(vocab_size, d_model)
        self.pos_embed = nn.Embedding(max_seq_len, d_model)
        self.embed_drop = nn.Dropout(dropout)
        self.embed_scale = math.sqrt(d_model)
        layer = TropicalEncoderLayer(d_model, nhead, dim_feedforward, dropout, lf_pieces,
                                     lf_mode, init_temp)
        return TropicalEncoder(layer, num_layers, norm=nn.LayerNorm(d_model))

    def _embed(self, input_ids: torch.Tensor,
               positions: Optional[torch.Tensor] = None) -> torch.Tensor:
        tok, pos = self.embed, self.pos_embed
        if (input_ids.is_cuda and input_ids.dtype in (torch.int32, torch.int64)
                and _plain_table(tok) and _plain_table(pos) and pos.padding_idx is None
                and input_ids.device == tok.weight.device == pos.weight.device
                and not _global_hooks()
                and not any(map(_transformed, (input_ids, tok.weight, pos.weight)))):
            ops.raise_seen_index_error(input_ids.device)      # of an earlier call
            return self.embed_drop(ops.embedding(input_ids, tok.weight, self.embed_scale,
                                                 pos_weight=pos.weight, positions=positions,
                                                 padding_idx=tok.padding_idx))
        if positions is None:
            positions = torch.arange(input_ids.shape[1], device=input_ids.device)[None]
        return self.embed_drop(self.embed(input_ids) * self.embed_scale +
                               self.pos_embed(positions))


class TropicalEncoderModel(_TokenModel):
    """Encoder-only (BERT-style) model (tropformer_dropin.py:616-663); attention_mask
    1 = keep, 0 = padding."""

    def __init__(self, vocab_size: int, d_model: int = 512, nhead: int = 8, num_layers: int = 6,
                 dim_feedforward: int = 2048, dropout: float = 0.1, max_seq_len: int = 512,
                 lf_pieces: int = 8, lf_mode: str = "blend", init_temp: float = 1.0):
        super().__init__()
        self.encoder = self._body(vocab_size, d_model, nhead, num_layers, dim_feedforward,
                                  dropout, max_seq_len, lf_pieces, lf_mode, init_temp)

    def forward(self, input_ids: torch.Tensor,
                attention_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        pad = (attention_mask == 0) if attention_mask is not None else None
        return self.encoder(self._embed(input_ids), src_key_padding_mask=pad)


class TropicalDecoderModel(_TokenModel):
    """Decoder-only (GPT-style) causal language model (tropformer_dropin.py:665-720)."""

    def __init__(self, vocab_size: int, d_model: int = 512, nhead: int = 8, num_layers: int = 6,
                 dim_feedforward: int = 2048, dropout: float = 0.1, max_seq_len: int = 2048,
                 lf_pieces: int = 8, lf_mode: str = "blend", init_temp: float = 1.0):
        super().__init__()
        self.layers = self._body(vocab_size, d_model, nhead, num_layers, dim_feedforward,
                                 dropout, max_seq_len, lf_pieces, lf_mode, init_temp)
        self.lm_head = nn.Linear(d_model, vocab_size, bias=False)

    def forward(self, input_ids: torch.Tensor,
                attention_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        mask = make_causal_mask(input_ids.shape[1], input_ids.device)
        pad = (attention_mask == 0) if attention_mask is not None else None
        x = self.layers(self._embed(input_ids), mask=mask, src_key_padding_mask=pad)
        return self.lm_head(x)

    @torch.no_grad()
    def generate(self, input_ids: torch.Tensor, max_new_tokens: int, *,
                 attention_mask: Optional[torch.Tensor] = None, temperature=1.0, top_k=0,
                 top_p=1.0, min_p=0.0, uniform: Optional[torch.Tensor] = None,
                 generator: Optional[torch.Generator] = None, page_size: int = 16,
                 keep: Optional[int] = None, recent: Optional[int] = None) -> torch.Tensor:
        """``max_new_tokens`` tokens [B, max_new_tokens] behind the prompts ``input_ids`` [B, L]
        (no reference counterpart), sampled as :func:`ops.sample_tokens` does (``temperature=0``:
        the best one).  ``attention_mask``: 1 = keep, 0 = padding, at the right of each row.
        ``uniform`` [max_new_tokens, B]: the random numbers, drawn from ``generator`` where None.

        ``keep``: a budget of cache slots for each sequence; a sequence over it by a page goes
        back to it, the last ``recent`` (None: a quarter) and those with the most accumulated
        attention weight staying.  Needs a CUDA device and a model in eval mode (or without
        dropout).  Under ``torch.autocast`` in bfloat16 the cache is of that type."""
        B, L = input_ids.shape
        if L < 1 or max_new_tokens < 1 or \
                L + max_new_tokens - 1 > self.pos_embed.num_embeddings:
            raise ValueError(f"{L} tokens and {max_new_tokens} new ones: needs at least one of "
                             f"each, within {self.pos_embed.num_embeddings} positions")
        if keep is not None and (keep < 1 or not 0 <= (recent or 0) <= keep):
            raise ValueError("keep must be at least 1 and recent from 0 to keep, got "
                             f"{keep} and {recent}")
        pad, counts = None, torch.full((B,), L, dtype=torch.int32, device=input_ids.device)
        if attention_mask is not None:
            live = attention_mask != 0
            if not bool(live[:, 0].all()) or bool((live[:, 1:] > live[:, :-1]).any()):
                raise ValueError("prompts must have a token and be padded at the right")
            pad, counts = ~live, live.sum(1, dtype=torch.int32)
        if uniform is None:
            uniform = torch.rand(max_new_tokens, B, device=input_ids.device, generator=generator)
        elif uniform.shape != (max_new_tokens, B):
            raise ValueError(f"uniform must be [{max_new_tokens}, {B}], got {tuple(uniform.shape)}")
        slots = L + max_new_tokens - 1
        if keep is not None:
            slots = min(slots, max(L, keep + page_size))
        attn = self.layers.layers[0].self_attn
        # keys and values come in the type of their projections
        dtype = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else \
            attn.k_proj.weight.dtype
        cache = TropicalPagedKVCache(len(self.layers.layers), B, attn.num_heads, attn.d_k, slots,
                                     page_size=page_size, collect_mass=keep is not None,
                                     dtype=dtype, device=input_ids.device)
        choices = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        cache.begin(counts, L)
        x = self.layers(self._embed(input_ids), mask=make_causal_mask(L, input_ids.device),
                        src_key_padding_mask=pad, cache=cache)
        x = x[torch.arange(B, device=x.device), counts.long() - 1]
        out = torch.empty(max_new_tokens, B, dtype=torch.int64, device=x.device)
        positions = counts.to(input_ids.dtype)[:, None]
        for t in range(max_new_tokens):
            out[t] = ops.sample_tokens(self.lm_head(x), uniform[t], **choices)
            if t + 1 == max_new_tokens:
                break
            if keep is not None and cache.most >= keep + page_size:
                cache.evict(keep, keep // 4 if recent is None else recent)
            cache.step()
            ids = out[t].to(input_ids.dtype)[:, None]
            x = self.layers(self._embed(ids, positions), cache=cache)[:, 0]
            positions = positions + 1
        return out.t().contiguous()


class TropicalViT(nn.Module):
    """Vision transformer on a tropical encoder (tropformer_dropin.py:739-797):
    patchify -> linear embedding -> CLS + learned positions -> encoder -> norm."""

    def __init__(self, img_size: int = 224, patch_size: int = 16, in_channels: int = 3,
                 d_model: int = 768, nhead: int = 12, num_layers: int = 12,
                 dim_feedforward: int = 3072, dropout: float = 0.1, lf_pieces: int = 8,
                 lf_mode: str = "blend", init_temp: float = 1.0):
        super().__init__()
        assert img_size % patch_size == 0
        self.patch_size = patch_size
        num_patches = (img_size // patch_size) ** 2
        self.patch_embed = nn.Linear(in_channels * patch_size * patch_size, d_model)
        nn.init.trunc_normal_(self.patch_embed.weight, std=0.02)
        self.cls_token = nn.Parameter(torch.zeros(1, 1, d_model))
        self.pos_embed = nn.Parameter(torch.zeros(1, num_patches + 1, d_model))
        nn.init.trunc_normal_(self.cls_token, std=0.02)
        nn.init.trunc_normal_(self.pos_embed, std=0.02)
        self.embed_drop = nn.Dropout(dropout)
        layer = TropicalEncoderLayer(d_model, nhead, dim_feedforward, dropout, lf_pieces,
                                     lf_mode, init_temp)
        self.encoder = TropicalEncoder(layer, num_layers, norm=nn.LayerNorm(d_model))

    def patchify(self, x: torch.Tensor) -> torch.Tensor:
        B, C, H, W = x.shape
        p = self.patch_size
        x = x.view(B, C, H // p, p, W // p, p).permute(0, 2, 4, 1, 3, 5).contiguous()
        return x.view(B, -1, C * p * p)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x = self.patch_embed(self.patchify(x))
        x = torch.cat([self.cls_token.expand(x.shape[0], -1, -1), x], dim=1)
        return self.encoder(self.embed_drop(x + self.pos_embed))


class TropicalViTForClassification(nn.Module):
    """TropicalViT plus a linear head on the CLS token (tropformer_dropin.py:800-819)."""

    def __init__(self, num_classes: int = 10, **vit_kwargs):
        super().__init__()
        self.vit = TropicalViT(**vit_kwargs)
        self.head = nn.Linear(vit_kwargs.get("d_model", 768), num_classes)
        nn.init.zeros_(self.head.bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.head(self.vit(x)[:, 0])

    def count_params(self) -> int:
        return sum(p.numel() for p in self.parameters() if p.requires_grad)


def maslov_summary(model: nn.Module) -> dict:
    """Per-head Maslov temperatures of every MaslovTemperature in ``model``."""
    return {name: m.temperatures.detach().cpu() for name, m in model.named_modules()
            if isinstance(m, tropical.MaslovTemperature)}


def lf_blend_summary(model: nn.Module) -> dict:
    """Mean sigmoid(blend_gate) of every blending LFDualActivation in ``model``."""
    return {name: torch.sigmoid(m.blend_gate).detach().cpu().mean().item()
            for name, m in model.named_modules()
            if isinstance(m, tropical.LFDualActivation) and hasattr(m, "blend_gate")}
