# Copyright 2026. Licensed under the Apache License, Version 2.0.
"""BERT-base encoder with a masked-LM head — for BASELINE config 5
(seqlen-512 hierarchical neighbor_allreduce). Standard architecture,
self-contained; uses torch's fused scaled_dot_product_attention, which on
ROCm lowers to the MIOpen/CK flash-attention path.

A batch can also be packed: its sequences one behind the other, without
padding, and ``cu_seqlens`` with their ends. Attention, norms and dropout then
run in bluefog_amd's own operators (ops/transformer.py), from the same modules:
each is called, with its own mode and probability, but for the ``nn.Dropout``,
whose masks the operators draw."""



import torch
import torch.nn as nn
import torch.nn.functional as F

__all__ = ["BertConfig", "BertForMaskedLM", "bert_base"]


class BertConfig:
    def __init__(
        self,
        vocab_size=30522,
        hidden_size=768,
        num_hidden_layers=12,
        num_attention_heads=12,
        intermediate_size=3072,
        max_position_embeddings=512,
        type_vocab_size=2,
        layer_norm_eps=1e-12,
        dropout=0.1,
    ):
        self.vocab_size = vocab_size
        self.hidden_size = hidden_size
        self.num_hidden_layers = num_hidden_layers
        self.num_attention_heads = num_attention_heads
        self.intermediate_size = intermediate_size
        self.max_position_embeddings = max_position_embeddings
        self.type_vocab_size = type_vocab_size
        self.layer_norm_eps = layer_norm_eps
        self.dropout = dropout


def _rate(dropout):
    """What a dropout module drops in its present mode."""
    if not isinstance(dropout, (nn.Dropout, nn.Identity)):
        raise TypeError(f"a packed batch takes nn.Dropout or nn.Identity, not {type(dropout).__name__}")
    return dropout.p if dropout.training and isinstance(dropout, nn.Dropout) else 0.0


class BertEmbeddings(nn.Module):
    def __init__(self, cfg: BertConfig):
        super().__init__()
        from bluefog_amd.ops.fused_modules import FusedAddLayerNorm

        self.word = nn.Embedding(cfg.vocab_size, cfg.hidden_size)
        self.position = nn.Embedding(cfg.max_position_embeddings, cfg.hidden_size)
        self.token_type = nn.Embedding(cfg.type_vocab_size, cfg.hidden_size)
        self.norm = FusedAddLayerNorm(cfg.hidden_size, eps=cfg.layer_norm_eps)
        self.dropout = nn.Dropout(cfg.dropout)
        self.register_buffer(
            "pos_ids", torch.arange(cfg.max_position_embeddings).unsqueeze(0), persistent=False
        )

    def forward(self, input_ids, cu_seqlens=None, seed=None):
        if cu_seqlens is not None:
            return self._packed(input_ids, cu_seqlens, seed)
        s = input_ids.shape[1]
        x = (
            self.word(input_ids)
            + self.position(self.pos_ids[:, :s])
            + self.token_type(torch.zeros_like(input_ids))
        )
        return self.dropout(self.norm(x))

    def _packed(self, input_ids, cu_seqlens, seed):
        from bluefog_amd.ops.transformer import counter_dropout

        token = torch.arange(input_ids.shape[0], device=input_ids.device, dtype=cu_seqlens.dtype)
        sequence = torch.searchsorted(cu_seqlens, token, right=True) - 1
        # rows behind the last sequence may lie further than the table goes, and
        # bounds on the GPU are not checked
        pos = (token - cu_seqlens[sequence]).clamp(0, self.position.num_embeddings - 1)
        x = self.word(input_ids) + self.position(pos) + self.token_type(torch.zeros_like(input_ids))
        x, p = self.norm(x, None, (0.0, None, 0)), _rate(self.dropout)
        return counter_dropout(x, p, seed) if p else x


class BertSelfAttention(nn.Module):
    def __init__(self, cfg: BertConfig):
        super().__init__()
        self.nh = cfg.num_attention_heads
        self.hd = cfg.hidden_size // cfg.num_attention_heads
        self.qkv = nn.Linear(cfg.hidden_size, 3 * cfg.hidden_size)
        self.out = nn.Linear(cfg.hidden_size, cfg.hidden_size)
        self.dropout_p = cfg.dropout

    def forward(self, x, cu_seqlens=None, seed=None, offset=0):
        if cu_seqlens is not None:
            return self._packed(x, cu_seqlens, seed, offset)
        B, S, H = x.shape
        qkv = self.qkv(x).reshape(B, S, 3, self.nh, self.hd).permute(2, 0, 3, 1, 4)
        q, k, v = qkv[0], qkv[1], qkv[2]
        o = F.scaled_dot_product_attention(
            q, k, v, dropout_p=self.dropout_p if self.training else 0.0
        )
        return self.out(o.transpose(1, 2).reshape(B, S, H))

    def _packed(self, x, cu_seqlens, seed, offset):
        from bluefog_amd.ops.transformer import packed_attention

        p = self.dropout_p if self.training else 0.0
        q, k, v = self.qkv(x).view(x.shape[0], 3, self.nh, self.hd).unbind(1)
        o = packed_attention(q, k, v, cu_seqlens, dropout_p=p, seed=seed, offset=offset)
        return self.out(o.flatten(1))


class BertLayer(nn.Module):
    def __init__(self, cfg: BertConfig):
        super().__init__()
        from bluefog_amd.ops.fused_modules import FusedAddLayerNorm

        self.attn = BertSelfAttention(cfg)
        # residual join + LayerNorm as one gfx950 kernel (eager off-GPU)
        self.norm1 = FusedAddLayerNorm(cfg.hidden_size, eps=cfg.layer_norm_eps)
        self.mlp = nn.Sequential(
            nn.Linear(cfg.hidden_size, cfg.intermediate_size),
            nn.GELU(),
            nn.Linear(cfg.intermediate_size, cfg.hidden_size),
        )
        self.norm2 = FusedAddLayerNorm(cfg.hidden_size, eps=cfg.layer_norm_eps)
        self.dropout = nn.Dropout(cfg.dropout)

    def forward(self, x, cu_seqlens=None, seed=None, offset=0):
        """On a packed batch the block's masks have offsets ``offset`` to
        ``offset + 2``."""
        if cu_seqlens is None:
            x = self.norm1(self.dropout(self.attn(x)), x)
            return self.norm2(self.dropout(self.mlp(x)), x)
        p = _rate(self.dropout)
        x = self.norm1(self.attn(x, cu_seqlens, seed, offset), x, (p, seed, offset + 1))
        return self.norm2(self.mlp(x), x, (p, seed, offset + 2))


class BertForMaskedLM(nn.Module):
    def __init__(self, cfg: BertConfig):
        super().__init__()
        self.cfg = cfg
        self.embeddings = BertEmbeddings(cfg)
        self.layers = nn.ModuleList(BertLayer(cfg) for _ in range(cfg.num_hidden_layers))
        self.head = nn.Linear(cfg.hidden_size, cfg.vocab_size, bias=False)
        self.head.weight = self.embeddings.word.weight  # weight tying
        self.apply(self._init)

    @staticmethod
    def _init(m):
        if isinstance(m, (nn.Linear, nn.Embedding)):
            nn.init.normal_(m.weight, std=0.02)
            if isinstance(m, nn.Linear) and m.bias is not None:
                nn.init.zeros_(m.bias)

    def forward(self, input_ids, labels=None, cu_seqlens=None):
        """``input_ids`` [batch, length], or [tokens] with ``cu_seqlens``
        (int32, 0 and the end of every sequence). A ``cu_seqlens`` on the CPU is
        checked and moved; one on the GPU is taken as it is, so that no step
        waits for it: its sequences have to fit the position table. Tokens
        behind the last sequence cost their share and mean nothing: label them
        -100."""
        if cu_seqlens is None:
            x = self.embeddings(input_ids)
            for layer in self.layers:
                x = layer(x)
        else:
            x = self._packed(input_ids, cu_seqlens)
        logits = self.head(x)
        if labels is not None:
            return F.cross_entropy(
                logits.view(-1, self.cfg.vocab_size), labels.view(-1), ignore_index=-100
            )
        return logits

    def _packed(self, input_ids, cu_seqlens):
        if input_ids.dim() != 1:
            raise ValueError("a packed batch is one row of tokens")
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
            raise ValueError("cu_seqlens has to be an int32 vector")
        if not cu_seqlens.is_cuda:
            ends = cu_seqlens.tolist()
            lengths = [b - a for a, b in zip(ends, ends[1:])]
            if ends[0] != 0 or ends[-1] > input_ids.shape[0] or any(n < 0 for n in lengths):
                raise ValueError("cu_seqlens has to rise from 0 to at most the number of tokens")
            if max(lengths, default=0) > self.cfg.max_position_embeddings:
                raise ValueError(
                    f"a sequence of {max(lengths)} tokens does not fit "
                    f"{self.cfg.max_position_embeddings} positions"
                )
            cu_seqlens = cu_seqlens.to(input_ids.device)
        # one seed for a step; every mask of it has an offset of its own
        drops = any(
            m.training and (m.dropout_p if isinstance(m, BertSelfAttention) else isinstance(m, nn.Dropout) and m.p)
            for m in self.modules()
        )
        seed = torch.randint(1 << 62, (1,), device=input_ids.device) if drops else None
        x = self.embeddings(input_ids, cu_seqlens, seed)
        for i, layer in enumerate(self.layers):
            x = layer(x, cu_seqlens, seed, 1 + 3 * i)
        return x


def bert_base():
    return BertForMaskedLM(BertConfig())
