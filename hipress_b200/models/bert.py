"""BERT-large (24 layers, hidden 1024, 16 heads, FFN 4096, vocab 30522) with a
masked-language-model head, for the onebit / CaSync-Ring configuration.

``fused=True`` runs the same parameters through the package's own layer operators
(:mod:`hipress_b200.ops.layers`): bias, GELU and residual in the products' epilogues, the
residual sum in the layer norm, attention without a copy of q, k and v.  On a GPU it wants
autocast (or 16-bit parameters), and no dropout of attention probabilities."""

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops import layer_norm, linear, self_attention


class BertConfig:
    """``attn_dropout``: of the attention probabilities (default: ``dropout``)."""

    def __init__(self, vocab_size=30522, hidden=1024, layers=24, heads=16, ffn=4096,
                 max_pos=512, type_vocab=2, dropout=0.1, attn_dropout=None, fused=False):
        self.vocab_size, self.hidden, self.layers, self.heads = vocab_size, hidden, layers, heads
        self.ffn, self.max_pos, self.type_vocab, self.dropout = ffn, max_pos, type_vocab, dropout
        self.attn_dropout = dropout if attn_dropout is None else attn_dropout
        self.fused = fused
        if fused and self.attn_dropout:
            raise ValueError("fused layers have no dropout of attention probabilities: attn_dropout=0")


def _norm(m, x, residual=None):
    return layer_norm(x, m.weight, m.bias, residual=residual, eps=m.eps)


class BertLayer(nn.Module):
    def __init__(self, c: BertConfig):
        super().__init__()
        self.heads = c.heads
        self.qkv = nn.Linear(c.hidden, 3 * c.hidden)
        self.proj = nn.Linear(c.hidden, c.hidden)
        self.ln1 = nn.LayerNorm(c.hidden, eps=1e-12)
        self.fc1 = nn.Linear(c.hidden, c.ffn)
        self.fc2 = nn.Linear(c.ffn, c.hidden)
        self.ln2 = nn.LayerNorm(c.hidden, eps=1e-12)
        self.drop = nn.Dropout(c.dropout)
        self.p = c.attn_dropout
        self.fused = c.fused

    def _add_norm(self, x, dense, norm, residual):
        """The layer norm of ``residual`` plus the dense layer's (dropped) result."""
        if self.training and self.drop.p:
            return _norm(norm, self.drop(linear(x, dense.weight, dense.bias)), residual)[0]
        return _norm(norm, linear(x, dense.weight, dense.bias, residual=residual))

    def _forward_fused(self, x, key_mask):
        B, S, H = x.shape
        qkv = linear(x, self.qkv.weight, self.qkv.bias).view(B, S, 3, self.heads, H // self.heads)
        x = self._add_norm(self_attention(qkv, key_mask=key_mask).view(B, S, H), self.proj, self.ln1, x)
        return self._add_norm(linear(x, self.fc1.weight, self.fc1.bias, activation="gelu"), self.fc2, self.ln2, x)

    def forward(self, x, key_mask=None):
        if self.fused:
            return self._forward_fused(x, key_mask)
        B, S, H = x.shape
        q, k, v = self.qkv(x).view(B, S, 3, self.heads, H // self.heads).permute(2, 0, 3, 1, 4)
        a = F.scaled_dot_product_attention(q, k, v, attn_mask=None if key_mask is None else key_mask[:, None, None],
                                           dropout_p=self.p if self.training else 0.0)
        a = a.transpose(1, 2).reshape(B, S, H)
        x = self.ln1(x + self.drop(self.proj(a)))
        return self.ln2(x + self.drop(self.fc2(F.gelu(self.fc1(x)))))


class BertForMaskedLM(nn.Module):
    def __init__(self, c: BertConfig | None = None):
        super().__init__()
        c = c or BertConfig()
        self.c = c
        self.tok = nn.Embedding(c.vocab_size, c.hidden)
        self.pos = nn.Embedding(c.max_pos, c.hidden)
        self.typ = nn.Embedding(c.type_vocab, c.hidden)
        self.ln = nn.LayerNorm(c.hidden, eps=1e-12)
        self.drop = nn.Dropout(c.dropout)
        self.layers = nn.ModuleList(BertLayer(c) for _ in range(c.layers))
        self.head_dense = nn.Linear(c.hidden, c.hidden)
        self.head_ln = nn.LayerNorm(c.hidden, eps=1e-12)
        self.head_bias = nn.Parameter(torch.zeros(c.vocab_size))
        self.apply(self._init)

    @staticmethod
    def _init(m):
        if isinstance(m, (nn.Linear, nn.Embedding)):
            nn.init.normal_(m.weight, 0.0, 0.02)
        if isinstance(m, nn.Linear) and m.bias is not None:
            nn.init.zeros_(m.bias)

    def forward(self, ids, labels=None, key_mask=None):
        """``key_mask`` [batch, length], bool: the positions that are no padding."""
        B, S = ids.shape
        fused = self.c.fused
        dense = linear if fused else F.linear
        pos = torch.arange(S, device=ids.device)
        x = self.tok(ids) + self.pos(pos)[None] + self.typ.weight[0][None, None]
        if fused and torch.is_autocast_enabled(x.device.type):
            x = x.to(torch.get_autocast_dtype(x.device.type))   # the layers keep the type of what they are given
        x = self.drop(_norm(self.ln, x) if fused else self.ln(x))
        for l in self.layers:
            x = l(x, key_mask)
        if fused:
            h = _norm(self.head_ln, linear(x, self.head_dense.weight, self.head_dense.bias, activation="gelu"))
        else:
            h = self.head_ln(F.gelu(self.head_dense(x)))
        if labels is None:
            return dense(h, self.tok.weight, self.head_bias)
        # score only the masked positions (labels == -100 elsewhere)
        sel = labels.view(-1) != -100
        hs = h.view(-1, h.shape[-1])[sel]
        logits = dense(hs, self.tok.weight, self.head_bias)
        return F.cross_entropy(logits.float(), labels.view(-1)[sel])


def bert_large(**kw):
    return BertForMaskedLM(BertConfig(**kw))


def bert_tiny(**kw):
    cfg = dict(vocab_size=1000, hidden=64, layers=2, heads=4, ffn=128, max_pos=64)
    cfg.update(kw)
    return BertForMaskedLM(BertConfig(**cfg))
