"""BERT encoder for MLM + NSP pre-training (Devlin et al. 2018).

``bert_large()``: 24 layers, hidden 1024, 16 heads, FFN 4096, vocab 30522,
512 positions (about 335 M parameters).  Attention goes through
``torch.nn.functional.scaled_dot_product_attention`` (a library kernel: the
model is the workload here, the gradient exchange is the product).

``activation_checkpoint="int8"`` keeps the inputs of the linear layers, the
GELU and the norms for the backward pass as 8-bit checkpoints
(``ops/act8.py``, ``ops/block_norm.py``): 33 bytes for 32 values in the place
of 64, or of 128 in fp32.  The forward pass computes the same, and the
parameters and their names are the same, so the option may change between
runs of one training.
"""

import torch
from torch import nn
import torch.nn.functional as F


EPS = 1e-12


def _is_int8(activation_checkpoint):
    if activation_checkpoint not in (None, "int8"):
        raise ValueError("activation_checkpoint: None or 'int8', not %r" % (activation_checkpoint,))
    return activation_checkpoint == "int8"


class BertLayer(nn.Module):
    """``residual_scale`` multiplies the residual stream before the block's output is added (DeepNorm); ``post_norm`` ("rms" or
    "layer") normalises the block's output first (sandwich norm); ``layer_scale`` (a number: the initial value) gives that output a
    learned gate for each channel."""

    def __init__(self, hidden, heads, ffn, dropout, activation_checkpoint=None, residual_scale=1.0, post_norm=None, layer_scale=None):
        super().__init__()
        self.heads = heads
        self.int8 = _is_int8(activation_checkpoint)
        self.residual_scale, self.post_norm = float(residual_scale), post_norm
        self.qkv = nn.Linear(hidden, 3 * hidden)
        self.proj = nn.Linear(hidden, hidden)
        self.ln1 = nn.LayerNorm(hidden, eps=EPS)
        self.fc1 = nn.Linear(hidden, ffn)
        self.fc2 = nn.Linear(ffn, hidden)
        self.ln2 = nn.LayerNorm(hidden, eps=EPS)
        self.drop = nn.Dropout(dropout)
        if post_norm not in (None, "rms", "layer"):
            raise ValueError("post_norm: None, 'rms' or 'layer', not %r" % (post_norm,))
        for i in (1, 2):
            norm = None if post_norm is None else (nn.RMSNorm if post_norm == "rms" else nn.LayerNorm)(hidden, eps=EPS)
            setattr(self, "post%d" % i, norm)
            setattr(self, "gate%d" % i, None if layer_scale is None else nn.Parameter(torch.full((hidden,), float(layer_scale))))

    def _join(self, x, block, ln, post, gate):
        """The stream after a block, normalised for the next one; with checkpoints also the Act8 of it."""
        block = self.drop(block)
        if self.int8:
            from ..ops.block_norm import residual_norm

            keep = torch.is_grad_enabled()      # (without a backward pass nothing reads a checkpoint)
            out = residual_norm(x, block, pre="layer", pre_weight=ln.weight, pre_bias=ln.bias, post=self.post_norm,
                                post_weight=None if post is None else post.weight, post_bias=getattr(post, "bias", None), gate=gate,
                                residual_scale=self.residual_scale, eps=EPS, return_stream=False, checkpoint_output=keep)
            return out if keep else (out, None)
        if post is not None:
            block = post(block)
        if gate is not None:
            block = block * gate
        return ln((x if self.residual_scale == 1.0 else self.residual_scale * x) + block), None

    def _linear(self, layer, x, held=None):
        if not self.int8:
            return layer(x)
        from ..ops import act8

        return act8.linear(x, layer.weight, layer.bias, checkpoint=held)

    def _gelu(self, x):
        """GELU, with checkpoints also the Act8 of it."""
        if not self.int8:
            return F.gelu(x), None
        from ..ops import act8

        if torch.is_grad_enabled():
            return act8.activation(x, "gelu", checkpoint_output=True)
        return act8.activation(x, "gelu"), None

    def forward(self, x, mask=None, held=None):
        """The new ``x``.  With ``activation_checkpoint="int8"`` the pair of it and its checkpoint (None without a backward pass), which the
        next layer takes as ``held``."""
        b, s, h = x.shape
        q, k, v = self._linear(self.qkv, x, held).view(b, s, 3, self.heads, h // self.heads).permute(2, 0, 3, 1, 4)
        a = F.scaled_dot_product_attention(q, k, v, attn_mask=mask)
        a = a.transpose(1, 2).reshape(b, s, h)
        x, held = self._join(x, self._linear(self.proj, a), self.ln1, self.post1, self.gate1)
        g, held = self._gelu(self._linear(self.fc1, x, held))
        x, held = self._join(x, self._linear(self.fc2, g, held), self.ln2, self.post2, self.gate2)
        return (x, held) if self.int8 else x


class BertForPreTraining(nn.Module):
    def __init__(self, vocab=30522, hidden=1024, layers=24, heads=16, ffn=4096, max_pos=512, type_vocab=2,
                 dropout=0.1, activation_checkpoint=None, residual_scale=1.0, post_norm=None, layer_scale=None):
        super().__init__()
        self.int8 = _is_int8(activation_checkpoint)
        self.tok = nn.Embedding(vocab, hidden)
        self.pos = nn.Embedding(max_pos, hidden)
        self.typ = nn.Embedding(type_vocab, hidden)
        self.ln = nn.LayerNorm(hidden, eps=EPS)
        self.drop = nn.Dropout(dropout)
        self.layers = nn.ModuleList(BertLayer(hidden, heads, ffn, dropout, activation_checkpoint, residual_scale, post_norm, layer_scale)
                                    for _ in range(layers))
        self.pooler = nn.Linear(hidden, hidden)
        self.mlm_dense = nn.Linear(hidden, hidden)
        self.mlm_ln = nn.LayerNorm(hidden, eps=EPS)
        self.mlm_bias = nn.Parameter(torch.zeros(vocab))
        self.nsp = nn.Linear(hidden, 2)
        self.apply(self._init)

    @staticmethod
    def _init(m):
        if isinstance(m, (nn.Linear, nn.Embedding)):
            nn.init.normal_(m.weight, std=0.02)
        if isinstance(m, nn.Linear) and m.bias is not None:
            nn.init.zeros_(m.bias)

    def forward(self, ids, token_type=None, mlm_labels=None, nsp_labels=None):
        b, s = ids.shape
        pos = torch.arange(s, device=ids.device).unsqueeze(0)
        if token_type is None:
            token_type = torch.zeros_like(ids)
        x = self.drop(self.ln(self.tok(ids) + self.pos(pos) + self.typ(token_type)))
        held = None
        for layer in self.layers:
            if self.int8:
                x, held = layer(x, held=held)
            else:
                x = layer(x)
        pooled = torch.tanh(self.pooler(x[:, 0]))
        if self.int8:
            from ..ops import act8

            h = self.mlm_ln(act8.activation(act8.linear(x, self.mlm_dense.weight, self.mlm_dense.bias, checkpoint=held), "gelu"))
        else:
            h = self.mlm_ln(F.gelu(self.mlm_dense(x)))
        logits = F.linear(h, self.tok.weight, self.mlm_bias)  # tied decoder
        nsp_logits = self.nsp(pooled)
        if mlm_labels is None:
            return logits, nsp_logits
        loss = F.cross_entropy(logits.view(-1, logits.size(-1)).float(), mlm_labels.view(-1), ignore_index=-100)
        if nsp_labels is not None:
            loss = loss + F.cross_entropy(nsp_logits.float(), nsp_labels)
        return loss


def bert_large(**kw):
    return BertForPreTraining(30522, 1024, 24, 16, 4096, 512, **kw)


def bert_tiny(**kw):
    return BertForPreTraining(1000, 64, 2, 4, 128, 64, **kw)
